// C[m][n] = sum_k A[m][k] B[n][k] on the 16-bit matrix instructions: the product every operator of this folder is made of.
//
// Operands.  Both are row-major with k contiguous, 16-byte aligned, a leading dimension that is a multiple of 8 elements, and hold one of
//   ONE plane   bf16 or fp16 numbers as they are
//   TWO planes  numbers of 22 bits: x = hi + lo, hi = fp16(x), lo = fp16(x - hi).  The planes lie interleaved, 32 k at a time: elements
//               [64 b, 64 b + 32) of a row are hi of k = 32 b .. 32 b + 31, the next 32 are lo of the same k.
// A product of TWO-plane operands is hi hi + hi lo + lo hi (lo lo is below 2^-22 of it): three fp16 matrix products give what fp32 ones give,
// at 2.5 PFLOP/s / 3 against 157 TFLOP/s of v_mfma_f32_16x16x4_f32.  Sums are fp32 in the accumulators in either case.  Values are scaled by a
// power of two that the caller chooses, so that hi never overflows and lo keeps its bits down to 2^-17 of the largest value.
//
// A tile is staged 128 bytes of every row at a time (64 k of ONE plane, 32 k of TWO): the interleaving makes both the same copy.  LDS-DMA,
// 16 bytes per lane; what lies outside the operand (rows past the end, k past the end) is an offset outside the buffer descriptor, which reads
// as zero.  A row's eight 16-byte pieces are stored in the order piece ^ (row / 2 mod 8): the 16 lanes of an operand read (16 rows, one piece)
// then touch each of the 64 banks once.
#pragma once
#include "../common.h"

namespace {

typedef unsigned short u16;
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

enum Planes { ONE = 1, TWO = 2 };
enum Element { BF16 = 0, FP16 = 1 };

__host__ __device__ static inline long long round_up(long long a, long long b) { return (a + b - 1) / b * b; }

// elements of a packed row that holds k numbers
__host__ __device__ static inline long long packed_width(int planes, long long k) { return planes == TWO ? 2 * round_up(k, 32) : round_up(k, 8); }
// place of number k in a packed row (its lo plane is 32 further); k, k + 1, .. of an aligned group of 32 are adjacent
__device__ __forceinline__ long long packed_at(int planes, long long k) { return planes == TWO ? (k >> 5) * 64 + (k & 31) : k; }

template <int EL> __device__ __forceinline__ u16 to_bits(float v) {
    if constexpr (EL == BF16) return __builtin_bit_cast(u16, (__bf16)v);
    else return __builtin_bit_cast(u16, (_Float16)v);
}
template <int EL> __device__ __forceinline__ float from_bits(u16 v) {
    if constexpr (EL == BF16) return (float)__builtin_bit_cast(__bf16, v);
    else return (float)__builtin_bit_cast(_Float16, v);
}

// one number into a packed row (p: the row's start)
template <int PL, int EL> __device__ __forceinline__ void pack1(u16* p, long long k, float v) {
    p += packed_at(PL, k);
    const u16 hi = to_bits<EL>(v);
    p[0] = hi;
    if constexpr (PL == TWO) p[32] = to_bits<EL>(v - from_bits<EL>(hi));
}
// four numbers k .. k + 3 (k a multiple of 4)
template <int PL, int EL> __device__ __forceinline__ void pack4(u16* p, long long k, f32x4 v) {
    p += packed_at(PL, k);
    u16 h[4], l[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        h[r] = to_bits<EL>(v[r]);
        l[r] = to_bits<EL>(v[r] - from_bits<EL>(h[r]));
    }
    *reinterpret_cast<u32x2*>(p) = u32x2{h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16};
    if constexpr (PL == TWO) *reinterpret_cast<u32x2*>(p + 32) = u32x2{l[0] | (unsigned)l[1] << 16, l[2] | (unsigned)l[3] << 16};
}
template <int PL, int EL> __device__ __forceinline__ f32x4 unpack4(const u16* p, long long k) {
    p += packed_at(PL, k);
    const u32x2 h = *reinterpret_cast<const u32x2*>(p);
    f32x4 v{from_bits<EL>((u16)h[0]), from_bits<EL>((u16)(h[0] >> 16)), from_bits<EL>((u16)h[1]), from_bits<EL>((u16)(h[1] >> 16))};
    if constexpr (PL == TWO) {
        const u32x2 l = *reinterpret_cast<const u32x2*>(p + 32);
        v += f32x4{from_bits<EL>((u16)l[0]), from_bits<EL>((u16)(l[0] >> 16)), from_bits<EL>((u16)l[1]), from_bits<EL>((u16)(l[1] >> 16))};
    }
    return v;
}

template <int EL> __device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
    if constexpr (EL == BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
        0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

struct Operand {
    const u16* p;          // element (0, 0)
    long long ld;          // elements from row to row
    int rows;
};

constexpr int kStageBytes = 128;                      // of every row
constexpr unsigned kOutside = 0x80000000u;            // an offset outside every descriptor

// A workgroup of WM x WN waves owns a BM x BN tile; a wave owns (BM / WM) x (BN / WN) of it.  acc[i][j] belongs to the wave's rows
// 16 i .. and columns 16 j ..; a lane holds row m = 16 i + (lane & 15) and the four columns n = 16 j + 4 (lane >> 4) ..  (the operands go to
// the instruction in the order B, A, so that the four values a lane holds are neighbours in a row of C).
template <int BM_, int BN_, int WM_, int WN_, int DEPTH_, int PL_, int EL_>
struct Tile {
    static constexpr int DEPTH = DEPTH_;                                     // stages in LDS
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, PL = PL_, EL = EL_;
    static constexpr int WAVES = WM * WN, THREADS = WAVES * 64, TM = BM / WM, TN = BN / WN, MI = TM / 16, NI = TN / 16;
    static constexpr int STAGE = (BM + BN) * kStageBytes;
    static constexpr int PITCH = BM + 8;                                      // of a row of the transposed tile (store_transposed)
    static constexpr int STAGES_LDS = DEPTH * STAGE, LDS = STAGES_LDS > BN * PITCH * 2 ? STAGES_LDS : BN * PITCH * 2;
    static constexpr int PER_CU = STAGES_LDS > 80 * 1024 ? 1 : STAGES_LDS > 40 * 1024 ? 2 : 4;               // workgroups that share a CU
    static constexpr int QA = BM / 8 / WAVES, QB = BN / 8 / WAVES;            // 1 KB copies (8 rows) of a wave per stage
    static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0 && WAVES % 2 == 0, "a wave copies whole groups of 8 rows");

    f32x4 acc[MI][NI];

    __device__ __forceinline__ static int wave() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }
    __device__ __forceinline__ static int row(int i) { return (wave() / WN) * TM + i * 16 + ((int)threadIdx.x & 15); }
    __device__ __forceinline__ static int col(int j) { return (wave() % WN) * TN + j * 16 + (((int)threadIdx.x & 63) >> 4) * 4; }

    // What the copies need of the tile that is worked on.
    byte_range range_a, range_b;
    unsigned at_a, at_b, step_a, step_b;
    int left;                                                                // packed elements behind the lane's piece of stage 0

    // copy q (of QA + QB) of stage t to the buffer `to`; a stage behind the last one is all zeros
    __device__ __forceinline__ void fetch(lds_address to, int t, int q) const {
        const bool in = t * 64 < left;
        const unsigned adv = (unsigned)t * kStageBytes;
        const int w = wave();
        if (q < QA) copy16_to_lds(range_a, to + (w + WAVES * q) * 1024, (in ? at_a : kOutside) + (adv + q * step_a));
        else copy16_to_lds(range_b, to + BM * kStageBytes + (w + WAVES * (q - QA)) * 1024, (in ? at_b : kOutside) + (adv + (q - QA) * step_b));
    }

    // Sets the copies of the first stages of a tile going.  k0, k1: the part of the packed width that is summed (k0 a multiple of 64); m0, n0: the
    // tile's corner.  Every wave of the workgroup calls this with the same arguments, when nobody uses the stages' LDS any more.
    __device__ __forceinline__ void start(const Operand& A, const Operand& B, int k0, int k1, int m0, int n0, char* lds) {
        const int w = wave(), lane = (int)threadIdx.x & 63;
        const int piece = (lane & 7) ^ (((4 * (w & 1)) + (lane >> 4)) & 7);          // of the row 8 q + lane / 8, q = w + WAVES i
        // The ranges end with the operand's (or the tile's) last row, so rows behind it read as zero by themselves.  (A tile spans at most
        // 256 rows of at most 2^21 numbers: its bytes stay below 2^31.)
        const int ra = A.rows - m0 < BM ? A.rows - m0 : BM, rb = B.rows - n0 < BN ? B.rows - n0 : BN;
        range_a = range_of(A.p + (long long)m0 * A.ld, (int)(ra * A.ld * 2));
        range_b = range_of(B.p + (long long)n0 * B.ld, (int)(rb * B.ld * 2));
        step_a = (unsigned)(8 * WAVES * A.ld * 2);
        step_b = (unsigned)(8 * WAVES * B.ld * 2);
        at_a = (unsigned)(((8 * w + (lane >> 3)) * A.ld + k0 + piece * 8) * 2);
        at_b = (unsigned)(((8 * w + (lane >> 3)) * B.ld + k0 + piece * 8) * 2);
        left = k1 - k0 - piece * 8;
        stages = (k1 - k0 + 63) / 64;
        const lds_address to = address_in_lds(lds);
#pragma unroll
        for (int t = 0; t < DEPTH; ++t)
#pragma unroll
            for (int q = 0; q < QA + QB; ++q) fetch(to + t * STAGE, t, q);
    }
    int stages;

    // The sums of the tile that was started.  The stages' LDS is free after the barrier that ends this.
    __device__ __forceinline__ void finish(char* lds) {
        const int w = wave(), lane = (int)threadIdx.x & 63;
        const lds_address lds0 = address_in_lds(lds);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

        // operand reads: row 16 i + (lane & 15) of the wave's part, piece 4 s + (lane >> 4) for s = 0, 1 (the two halves of 64 k; hi and lo)
        const int swz = ((lane & 15) >> 1) & 7, pc = lane >> 4;
        const int base_a = ((w / WN) * TM + (lane & 15)) * kStageBytes, base_b = BM * kStageBytes + ((w % WN) * TN + (lane & 15)) * kStageBytes;
        const int p0 = ((pc) ^ swz) * 16, p1 = ((pc + 4) ^ swz) * 16;

        // The operand reads of one half of a stage and the copies of the stage after the next run under the matrix instructions, a few behind every
        // row of the wave's part: issued together they would fill their queues and hold up the wave.  No wave waits for LDS or memory but at
        // the one barrier of a stage, by which its reads of stage t have arrived, its copies of stage t + 1 are in LDS (they had DEPTH - 1
        // stages' time), and the buffer of stage t may be written again.
        uint4 a0[MI], b0[NI], a1[MI], b1[NI];
        constexpr int READS = MI + NI, EACH_READ = (READS + MI - 2) / (MI - 1), EACH_COPY = (QA + QB + MI - 1) / MI;
        auto read = [&](uint4* a, uint4* b, const char* s, int p, int r) {                      // read r of READS
            if (r < NI) b[r] = *reinterpret_cast<const uint4*>(s + base_b + p + r * 16 * kStageBytes);
            else a[r - NI] = *reinterpret_cast<const uint4*>(s + base_a + p + (r - NI) * 16 * kStageBytes);
        };
        auto multiply = [&](const uint4* a, const uint4* b, int i) {
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = mfma16<EL>(b[j], a[i], acc[i][j]);
        };
        // (what a wave issues arrives in order: all but the copies of the stages behind this one, or what was issued behind them)
        vm_wait<(DEPTH - 1) * (QA + QB)>();
        __builtin_amdgcn_s_barrier();
#pragma unroll
        for (int r = 0; r < READS; ++r) read(a0, b0, lds, p0, r);
        int here = 0;                                                        // the buffer of stage t
        for (int t = 0; t < stages; ++t) {
            const int there = here + STAGE == STAGES_LDS ? 0 : here + STAGE;
            const char* s = lds + here;
            const char* next = lds + there;
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int r = i * EACH_READ; r < (i + 1) * EACH_READ && r < READS; ++r) read(a1, b1, s, p1, r);
                multiply(a0, b0, i);
            }
            if constexpr (PL == TWO) {                                       // hi hi, hi lo; then lo hi
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < MI; ++i) multiply(a0, b1, i);
            }
            __builtin_amdgcn_sched_barrier(0);
            UNFLOW_WAIT_LGKMCNT0();
            vm_wait<(DEPTH - 2) * (QA + QB)>();
            __builtin_amdgcn_s_barrier();
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int q = i * EACH_COPY; q < (i + 1) * EACH_COPY && q < QA + QB; ++q) fetch(lds0 + here, t + DEPTH, q);
#pragma unroll
                for (int r = i * EACH_READ; r < (i + 1) * EACH_READ && r < READS; ++r) read(a0, PL == TWO ? b1 : b0, next, p0, r);
                multiply(a1, PL == TWO ? b0 : b1, i);
            }
            if constexpr (PL == TWO) {
#pragma unroll
                for (int j = 0; j < NI; ++j) b0[j] = b1[j];
            }
            here = there;
        }
        UNFLOW_WAIT_VMCNT0();
        __syncthreads();
    }
    __device__ __forceinline__ void run(const Operand& A, const Operand& B, int k0, int k1, int m0, int n0, char* lds) {
        start(A, B, k0, k1, m0, n0, lds);
        finish(lds);
    }

    // The transpose of the tile, value(i, j) being the four numbers that belong to acc[i][j], into packed rows: dst row n holds the numbers of
    // column n at k = m.  A lane's four numbers lie in four dst rows; through LDS (half of m at a time for TWO planes) the rows leave in 16-byte
    // pieces.  `width`: elements of a dst row; LDS is free when this is called and not when it returns.  AS: what the numbers become.
    template <int AS = EL, class F>
    __device__ __forceinline__ void store_transposed(char* lds, u16* __restrict__ dst, long long ld, int rows, long long width, int m0, int n0,
        F&& value) {
        static_assert(WM == 2, "the halves of m are the wave rows");
        constexpr int R = BM / PL;
        u16* s = reinterpret_cast<u16*>(lds);
#pragma unroll
        for (int pass = 0; pass < PL; ++pass) {
            if (PL == 1 || wave() / WN == pass) {
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int j = 0; j < NI; ++j) {
                        const f32x4 v = value(i, j);
#pragma unroll
                        for (int r = 0; r < 4; ++r) pack1<PL, AS>(s + (col(j) + r) * PITCH, row(i) - pass * R, v[r]);
                    }
            }
            __syncthreads();
            const long long first = packed_at(PL, m0 + pass * R);
            for (int c = (int)threadIdx.x; c < BN * BM / 8; c += THREADS) {
                const int n = c / (BM / 8), e = c % (BM / 8) * 8;
                u16* to = dst + (long long)(n0 + n) * ld + first + e;
                if (n0 + n < rows && first + e < width) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(s + n * PITCH + e);
            }
            if (pass + 1 < PL) __syncthreads();
        }
    }
};

// Order of the tiles of an mt x nt grid: workgroups of one XCD take neighbouring tiles, and these go down groups of 8 tile rows before the next
// tile column, so that what runs at one time shares operand rows in the XCD's L2.
__device__ __forceinline__ void tile_of(int id, int mt, int nt, int& tm, int& tn) {
    const int group = 8 * nt, g = id / group, first = g * 8;
    const int size = mt - first < 8 ? mt - first : 8, in = id - g * group;
    tm = first + in % size;
    tn = in / size;
}

// ---- packing an operand
template <class T> __device__ __forceinline__ float load1(const T* p);
template <> __device__ __forceinline__ float load1<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float load1<__bf16>(const __bf16* p) { return (float)*p; }
template <> __device__ __forceinline__ float load1<_Float16>(const _Float16* p) { return (float)*p; }

template <class T> __device__ __forceinline__ void store4(T* p, f32x4 v, int n) {            // n = 1 .. 4 of the four values
    if (n == 4 && ((size_t)p & (4 * sizeof(T) - 1)) == 0) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(p) = v;
        else {
            u16 h[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) h[r] = __builtin_bit_cast(u16, (T)v[r]);
            *reinterpret_cast<u32x2*>(p) = u32x2{h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16};
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r < n) p[r] = (T)v[r];
    }
}

}  // namespace
