// Softmax cross entropy of z = scale * H W^T (H [N, D] hidden rows, W [V, D] one row per class) without ever holding z, and its gradients.
//
//   forward    loss_i = lse_i - z_i,t(i),  lse_i = log sum_v exp(z_iv)
//              A tile of z lives in the accumulators of the product only.  Of each of its rows the running maximum and the sum of the
//              exponentials leave the tile (8 bytes per row and tile), a second kernel joins them over the tiles, in fixed order.
//   backward   dH = G W,  dW = G^T H,  G_iv = g_i scale (exp(z_iv - lse_i) - [v = t(i)])
//              in pieces of the classes: a piece of G is recomputed from H, W and lse, held in 16 bits (both ways round, since the two products
//              contract its two sides), and used up by both products before the next piece.  dW of a piece is complete; dH gathers in fp32.
//
// What bounds it: the matrix products, 2 N V D operations forward and 8 N V D for the three of the backward pass with z recomputed (6 N V D
// where z could be kept); reading W bounds the forward pass of few rows.  Numbers: 16-bit inputs go to the matrix instructions as they are;
// fp32 inputs as two fp16 planes scaled by the largest magnitude (mfma16.h).  G is held in fp16 (two planes for fp32) times 2^14: 11 (22) bits of
// every probability down to 2^-28 (2^-17).  For bf16 inputs its own 8 bits would do as far as the products go, but where a gradient's sum cancels
// they show: 9246 rows against 9246 classes of 32, scale 14, came out 1.6 times as far off as the rounding of the gradients to bf16 alone.  The
// other operands of these products, transposes that are written anyhow, are then fp16 as well, times the power of two that brings the largest
// magnitude to [2^14, 2^15); to find it bf16 inputs are read once more.  The uniform factors of G (scale, the upstream gradient of a reduced loss)
// are applied to the sums.
//
// A row whose target is `ignore_index` has loss 0 and no gradient, whatever its hidden row holds (it is left out of the largest magnitude, and
// enters the transposed H as zeros: 0 * NaN never meets a sum).  Any other target outside [0, V) makes its row's loss and gradients NaN.
#include "pack.h"
#include "plan.h"
#include <cmath>
#include <cstring>

namespace {

constexpr int kFp32 = 0, kBf16 = 1, kFp16 = 2;                     // UNFLOW_DTYPE_*
constexpr int kMaxima = 1024;                                      // workgroups at most that pack one input, each noting the largest magnitude it met

// fp32 rows are packed with a power of two of their own that brings the row's largest magnitude to [2^14, 2^15), their transposes (where rows are
// what is summed over) with one for the whole matrix.
struct Exponents { int h, w; };      // of the transposes
// of a row: log2(e) max z, 1 / sum exp(z - max z), sum over all classes but the target times that
struct Row { float top, inverse, others, unused; };

__device__ __forceinline__ float finite_magnitude(float m, f32x4 v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float a = fabsf(v[k]);
        m = a <= 3.4028235e38f ? fmaxf(m, a) : m;
    }
    return m;
}
__device__ __forceinline__ float wave_largest(float m) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    return m;
}
__device__ __forceinline__ int exponent_for(float largest) { return largest > 0.f ? 14 - ilogbf(largest) : 0; }

// H and W into packed rows, one launch: the first `blocks_h` workgroups take H (0: H needs no packing), the rest W; a wave takes a row at a time.
// fp32: the rows' exponents, and the workgroups' largest finite magnitudes of the rows that count (maxima [2][kMaxima]).  Bound by bytes: 11020 rows
// of 777 fp32 numbers 25 us (34 MB read, 35 written).
struct Packed { u16 *h, *w; int *eh, *ew; float* maxima; };
template <class T, int PL, int EL>
__global__ __launch_bounds__(256) void pack_inputs_kernel(Source h, Source w, int blocks_h, Packed to, long long ldd, int width) {
    __shared__ float red[4];
    const bool second = (int)blockIdx.x >= blocks_h;
    const Source s = second ? w : h;
    u16* dst = second ? to.w : to.h;
    const int block = (int)blockIdx.x - (second ? blocks_h : 0), blocks = second ? (int)gridDim.x - blocks_h : blocks_h;
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    float all = 0.f;
    for (int first = block * 4; first < s.rows; first += blocks * 4) {
        const int r = first + wave < s.rows ? first + wave : s.rows - 1;                  // (waves past the last row repeat it)
        const T* row = (const T*)s.p + (long long)r * s.ld;
        int e = 0;
        if constexpr (PL == TWO) {
            float m = 0.f;
            for (int k = lane * 4; k < s.cols; k += 256) m = finite_magnitude(m, load4(row + k, s.cols - k));
            m = wave_largest(m);
            e = exponent_for(m);
            if (!(s.label && s.label[r] == s.skip)) all = fmaxf(all, m);
            if (lane == 0) (second ? to.ew : to.eh)[r] = e;
        }
        for (int k = lane * 4; k < width; k += 256) pack4<PL, EL>(dst + r * ldd, k, scaled(load4(row + k, s.cols - k), e));
    }
    if constexpr (PL == TWO) {
        if (lane == 0) red[wave] = all;
        __syncthreads();
        if (threadIdx.x == 0) to.maxima[(second ? kMaxima : 0) + block] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    }
}

// log2(e) z of an accumulator of row m and column n: exponentials are then single instructions
constexpr float kLog2E = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }
struct Logits { float scale; const int *eh, *ew; };             // scale: of the loss, times log2(e)
template <int PL> __device__ __forceinline__ f32x4 logits_of(const Logits& l, f32x4 acc, int eh, int n, int last) {
    acc *= l.scale;
    if constexpr (PL == TWO) {
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = ldexpf(acc[r], -(eh + l.ew[n + r < last ? n + r : last]));
    }
    return acc;
}

// ---- forward: of each row of a tile of z the maximum (times log2(e), as all that follows) and the sum of exp(z - maximum) over the classes that
// are not the row's target, and the target's z.  partial [tile column][N].  Bound by the matrix instructions, and for short rows by what a tile's
// end costs: 8192 rows, 131072 classes of 4096 bf16 6.3 ms = 1400 TFLOP/s; 4096, 32000 of 2048 470 to 490 us = 1100 to 1140; fp32 1013, 10007 of 777
// 56 us = 280.
template <class TileT>
__global__ __launch_bounds__(TileT::THREADS, 2) void lce_forward_kernel(Operand H, Operand W, int width, Logits how,
        const long long* __restrict__ target, float2* __restrict__ partial, float* __restrict__ ztarget) {
    UNFLOW_DYNAMIC_LDS(char, lds);
    const int mt = ceil_div(H.rows, TileT::BM), nt = ceil_div(W.rows, TileT::BN), total = mt * nt;
    float2* rows = reinterpret_cast<float2*>(lds + TileT::STAGES_LDS);                    // [WN][BM]
    const int wn = TileT::wave() % TileT::WN, group = ((int)threadIdx.x & 63) >> 4;
    int id = (int)blockIdx.x, tm, tn;
    tile_of(xcd_remap(id, total), mt, nt, tm, tn);
    TileT T;
    T.start(H, W, 0, width, tm * TileT::BM, tn * TileT::BN, lds);
    // A workgroup goes through tiles a grid apart: the copies of the next one are under way while this one's sums are dealt with (4 % of 4096 rows,
    // 32000 classes of 2048).
    for (bool more = true; more;) {
        T.finish(lds);
        const int m0 = tm * TileT::BM, n0 = tn * TileT::BN, column = tn;
        id += (int)gridDim.x;
        more = id < total;
        if (more) {
            tile_of(xcd_remap(id, total), mt, nt, tm, tn);
            T.start(H, W, 0, width, tm * TileT::BM, tn * TileT::BN, lds);
        }
        const bool edge = n0 + TileT::BN > W.rows;
#pragma unroll
        for (int i = 0; i < TileT::MI; ++i) {
            const int m = m0 + TileT::row(i);
            const long long t = m < H.rows ? target[m] - n0 : -1;                        // the target's place in this tile
            const int own = t >= 0 && t < TileT::BN && t + n0 < W.rows ? (int)t : -1, eh = TileT::PL == TWO && m < H.rows ? how.eh[m] : 0;
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < TileT::NI; ++j) {
                f32x4 z = logits_of<TileT::PL>(how, T.acc[i][j], eh, n0 + TileT::col(j), W.rows - 1);
                if (edge)
#pragma unroll
                    for (int r = 0; r < 4; ++r) z[r] = n0 + TileT::col(j) + r < W.rows ? z[r] : -INFINITY;
                T.acc[i][j] = z;
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, z[r]);
            }
            // (few of a wave's rows have their target among its columns)
            if (__ballot(own >= 0))
#pragma unroll
                for (int j = 0; j < TileT::NI; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (TileT::col(j) + r == own) {
                            ztarget[m] = T.acc[i][j][r];
                            T.acc[i][j][r] = -INFINITY;
                        }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float base = top == -INFINITY ? 0.f : top;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < TileT::NI; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) sum += exp2_of(T.acc[i][j][r] - base);
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            if (group == 0) rows[wn * TileT::BM + TileT::row(i)] = make_float2(top, sum);
        }
        __syncthreads();
        for (int r = (int)threadIdx.x; r < TileT::BM && m0 + r < H.rows; r += TileT::THREADS) {
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int q = 0; q < TileT::WN; ++q) top = fmaxf(top, rows[q * TileT::BM + r].x);
#pragma unroll
            for (int q = 0; q < TileT::WN; ++q) {
                const float2 v = rows[q * TileT::BM + r];
                // (without a maximum: 0, or NaN from NaNs, which fmaxf passes over)
                sum += v.x != -INFINITY ? v.y * exp2_of(v.x - top) : v.y;
            }
            partial[(long long)column * H.rows + m0 + r] = make_float2(top, sum);
        }
    }
}

// ---- forward of few rows (at most 16 NF): reading W is all there is to it (one row, 32000 classes of 2048 bf16: 23 us = 5.7 TB/s).  Where the tiles
// above could take W as it is, 16 rows go here: beyond, the four waves of a tile share the rows of H (61 rows against 50257 classes of 1024 fp16: 20
// us there, 36 here).  Where W would have to be packed first, written and read once more, 64 rows of fp32 (50257 classes of 1023, whole calls: 1 row
// 52 us, 64 rows 125, 65 rows by the tiles 214) and 32 of 16-bit numbers, which loads off 4 bytes slow down (the same in fp16: 1 row 55 us, 32 rows
// 94, by the tiles 89; 59332 of 755: 40, 72, 78; 14068 of 1235: 20, 32, 42).  A workgroup takes 16 CF classes, its four waves a quarter of D each,
// AHEAD steps of loads in flight; the rows of W go from memory to the matrix instruction as they lie there.  16-bit numbers: 32 k a step, lane l
// holds k = 8 (l >> 4) .. of row l & 15.  fp32: 16 k a step as four v_mfma_f32_16x16x4_f32, the e-th taking k = 4 (l >> 4) + e -- fp32 arithmetic
// throughout, and no packing.
// Rows need no alignment: a lane's 16 bytes are loaded from where they lie, and the last ones of a row as its last 16 bytes, of which both operands
// drop what the lane before has taken already (the order of k does not matter as long as both agree).
template <class T> struct Few {
    static constexpr int EACH = 16 / sizeof(T), STEP = 4 * EACH;
    struct Piece { unsigned v[4]; } __attribute__((packed, aligned(sizeof(T))));
    __device__ __forceinline__ static uint4 load(const T* p) {
        const Piece q = *reinterpret_cast<const Piece*>(p);
        return uint4{q.v[0], q.v[1], q.v[2], q.v[3]};
    }
    // without the first `skip` numbers
    __device__ __forceinline__ static uint4 behind(uint4 q, int skip) {
        unsigned v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) v[i] = i < skip ? 0u : v[i];
            else v[i] = 2 * i + 1 < skip ? 0u : 2 * i < skip ? v[i] & 0xffff0000u : v[i];
        }
        return uint4{v[0], v[1], v[2], v[3]};
    }
};
template <class T> __device__ __forceinline__ f32x4 few_product(uint4 a, uint4 b, f32x4 c) {
    if constexpr (sizeof(T) == 4) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
        return c;
    } else return mfma16<__is_same(T, __bf16) ? BF16 : FP16>(a, b, c);
}
template <class T, int NF, int CF, int AHEAD>
__global__ __launch_bounds__(256) void lce_few_kernel(const T* __restrict__ H, long long ldh, const T* __restrict__ W, long long ldw, int N, int V,
        int D, float scale, const long long* __restrict__ target, float2* __restrict__ partial, float* __restrict__ ztarget) {
    constexpr int ROWS = 16 * NF, PER = 256 / ROWS, CLASSES = 16 * CF / PER, PITCH = 16 * CF + 2;
    __shared__ float sums[4][ROWS][PITCH];
    const int lane = (int)threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int v0 = (int)blockIdx.x * 16 * CF, k_lane = (lane >> 4) * Few<T>::EACH, r_lane = lane & 15;
    const T* wrow[CF];
    const T* hrow[NF];
    // (classes behind the last repeat it, unused)
#pragma unroll
    for (int c = 0; c < CF; ++c) wrow[c] = W + (long long)(v0 + 16 * c + r_lane < V ? v0 + 16 * c + r_lane : V - 1) * ldw;
#pragma unroll
    for (int i = 0; i < NF; ++i) hrow[i] = H + (long long)(16 * i + r_lane < N ? 16 * i + r_lane : N - 1) * ldh;
    f32x4 acc[CF][NF];
#pragma unroll
    for (int c = 0; c < CF; ++c)
#pragma unroll
        for (int i = 0; i < NF; ++i) acc[c][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int steps = ceil_div(D, Few<T>::STEP);
    for (int first = 0; first < steps; first += 4 * AHEAD) {
        uint4 a[AHEAD][CF], b[AHEAD][NF];
        int skip[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            // (a wave takes two steps in a row: whole lines of W)
            const int k = (first + (u / 2) * 8 + w * 2 + u % 2) * Few<T>::STEP + k_lane, from = k < D - Few<T>::EACH ? k : D - Few<T>::EACH;
            skip[u] = k - from;
#pragma unroll
            for (int c = 0; c < CF; ++c) a[u][c] = Few<T>::load(wrow[c] + from);
#pragma unroll
            for (int i = 0; i < NF; ++i) b[u][i] = Few<T>::load(hrow[i] + from);
        }
        if ((first + 4 * AHEAD) * Few<T>::STEP > D)                      // (a row's end is in reach)
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
#pragma unroll
                for (int c = 0; c < CF; ++c) a[u][c] = Few<T>::behind(a[u][c], skip[u]);
#pragma unroll
                for (int i = 0; i < NF; ++i) b[u][i] = Few<T>::behind(b[u][i], skip[u]);
            }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int c = 0; c < CF; ++c)
#pragma unroll
                for (int i = 0; i < NF; ++i) acc[c][i] = few_product<T>(a[u][c], b[u][i], acc[c][i]);
    }
    // a lane holds row 16 i + (lane & 15), classes 16 c + 4 (lane >> 4) ..
#pragma unroll
    for (int c = 0; c < CF; ++c)
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) sums[w][16 * i + r_lane][16 * c + 4 * (lane >> 4) + r] = acc[c][i][r];
    __syncthreads();
    const int m = (int)threadIdx.x / PER, part = (int)threadIdx.x % PER;
    const long long t = m < N ? target[m] : -1;
    float z[CLASSES], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int c = 0; c < CLASSES; ++c) {
        const int at = part + PER * c, n = v0 + at;
        z[c] = n < V ? ((sums[0][m][at] + sums[1][m][at]) + (sums[2][m][at] + sums[3][m][at])) * scale : -INFINITY;
        top = fmaxf(top, z[c]);
        if (n == t && n < V) {
            ztarget[m] = z[c];
            z[c] = -INFINITY;
        }
    }
#pragma unroll
    for (int o = PER / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int c = 0; c < CLASSES; ++c) sum += exp2_of(z[c] - base);
#pragma unroll
    for (int o = PER / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (part == 0 && m < N) partial[(long long)blockIdx.x * N + m] = make_float2(top, sum);
}

// two (maximum, sum) pairs as one
__device__ __forceinline__ float2 joined(float2 x, float2 y) {
    const float both = fmaxf(x.x, y.x), base = both == -INFINITY ? 0.f : both;
    return make_float2(both, x.y * (x.x == -INFINITY ? 1.f : exp2_of(x.x - base)) + y.y * (y.x == -INFINITY ? 1.f : exp2_of(y.x - base)));
}
// the pairs of row m of the tiles first, first + step, ..; the loads of eight are under way together
__device__ __forceinline__ float2 joined_tiles(const float2* __restrict__ partial, int first, int step, int tiles, int N, int m) {
    float2 pair = make_float2(-INFINITY, 0.f);
    for (int t = first; t < tiles; t += 8 * step) {
        float2 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = t + k * step < tiles ? partial[(long long)(t + k * step) * N + m] : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) pair = joined(pair, v[k]);
    }
    return pair;
}
// A row's statistics and loss from its joined pair.  The target's own term joins here: where it outweighs the others, loss = log1p(others / own)
// and others / all = 1 - p keep the digits that 1 - p would lose.
__device__ __forceinline__ float row_of(float2 pair, long long t, long long ignore, int V, const float* __restrict__ ztarget,
        Row* __restrict__ stats) {
    const float base = pair.x == -INFINITY ? 0.f : pair.x, others = pair.y;
    const bool known = t >= 0 && t < V;
    const float zt = known ? *ztarget : -INFINITY, own = known ? exp2_of(zt - base) : 0.f, all = others + own;
    *stats = Row{base, 1.f / all, others / all, 0.f};
    return t == ignore ? 0.f : !known ? NAN : own > 0.01f * others ? log1pf(others / own) : (base - zt) * kLn2 + logf(all);
}

// the tiles' pairs of a row joined in fixed order: R rows x 256 / R shares of the tiles per workgroup.  4 to 10 us: the latency of a launch and
// of its loads
template <int R>
__global__ __launch_bounds__(256) void lce_join_kernel(const float2* __restrict__ partial, int tiles, int N, int V,
        const long long* __restrict__ target, long long ignore, const float* __restrict__ ztarget, Row* __restrict__ stats,
        float* __restrict__ losses) {
    constexpr int SHARES = 256 / R;
    __shared__ float2 part[SHARES][R + 1];
    const int r = threadIdx.x % R, share = threadIdx.x / R, m = blockIdx.x * R + r;
    part[share][r] = m < N ? joined_tiles(partial, share, SHARES, tiles, N, m) : make_float2(-INFINITY, 0.f);
    __syncthreads();
    for (int half = SHARES / 2; half > 0; half /= 2) {
        if (share < half) part[share][r] = joined(part[share][r], part[share + half][r]);
        __syncthreads();
    }
    if (share == 0 && m < N) losses[m] = row_of(part[0][r], target[m], ignore, V, ztarget + m, stats + m);
}

// loss = sum of a thread's losses over the workgroup (mean: divided by the number of rows that are not ignored, at least 1, which is left for the
// backward pass); fixed order
__device__ __forceinline__ void reduce_losses(float s, float c, int mean, float* __restrict__ loss, float* __restrict__ count) {
    __shared__ float red[16], cnt[16];
    s = wave_sum(s);
    c = wave_sum(c);
    if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = s; cnt[threadIdx.x >> 6] = c; }
    __syncthreads();
    if (threadIdx.x == 0) {
        s = c = 0.f;
        for (int q = 0; q < 16; ++q) { s += red[q]; c += cnt[q]; }
        count[0] = fmaxf(c, 1.f);
        loss[0] = mean ? s / fmaxf(c, 1.f) : s;
    }
}
__global__ __launch_bounds__(1024) void lce_reduce_kernel(const float* __restrict__ losses, const long long* __restrict__ target, long long ignore,
        int N, int mean, float* __restrict__ loss, float* __restrict__ count) {
    float s = 0.f, c = 0.f;
    for (int i = threadIdx.x; i < N; i += 1024) {
        s += losses[i];
        c += target[i] != ignore ? 1.f : 0.f;
    }
    reduce_losses(s, c, mean, loss, count);
}
// both at once for up to 1024 rows of few tiles: a launch less where launches are what a pass costs
__global__ __launch_bounds__(1024) void lce_join_reduce_kernel(const float2* __restrict__ partial, int tiles, int N, int V,
        const long long* __restrict__ target, long long ignore, const float* __restrict__ ztarget, Row* __restrict__ stats, int mean,
        float* __restrict__ loss, float* __restrict__ count) {
    const int m = threadIdx.x;
    float s = 0.f, c = 0.f;
    if (m < N) {
        const long long t = target[m];
        s = row_of(joined_tiles(partial, 0, 1, tiles, N, m), t, ignore, V, ztarget + m, stats + m);
        c = t != ignore ? 1.f : 0.f;
    }
    reduce_losses(s, c, mean, loss, count);
}

// ---- backward
// The largest finite magnitudes that workgroups meet in bf16 inputs as pack_inputs_kernel notes them for fp32 ones (rows of 16-byte pieces, zeros
// behind the last number).  A wave takes a row at a time, four pieces a lane under way together.  Bound by bytes: 139264 rows of 4096
// 183 us = 6.2 TB/s.
__global__ __launch_bounds__(256) void lce_magnitudes_kernel(Operand h, Operand w, int pieces, int blocks_h, const long long* __restrict__ target,
        long long ignore, float* __restrict__ maxima) {
    __shared__ unsigned red[4];
    const bool second = (int)blockIdx.x >= blocks_h;
    const Operand s = second ? w : h;
    const int block = (int)blockIdx.x - (second ? blocks_h : 0), blocks = second ? (int)gridDim.x - blocks_h : blocks_h;
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    unsigned top = 0;                                                    // magnitudes of bf16 numbers order as their bits
    auto meet = [&](unsigned bits) { top = bits < 0x7f80u && bits > top ? bits : top; };
    for (int r = block * 4 + wave; r < s.rows; r += blocks * 4) {
        if (!second && target[r] == ignore) continue;
        const uint4* row = reinterpret_cast<const uint4*>(s.p + (long long)r * s.ld);
        for (int k = lane; k < pieces; k += 256) {
            uint4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = k + 64 * u < pieces ? row[k + 64 * u] : uint4{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const unsigned e[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    meet(e[i] & 0x7fffu);
                    meet(e[i] >> 16 & 0x7fffu);
                }
            }
        }
    }
    const float all = wave_largest(__builtin_bit_cast(float, top << 16));
    if (lane == 0) red[wave] = __builtin_bit_cast(unsigned, all);        // (positive floats order as their bits)
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int q = 1; q < 4; ++q) red[0] = red[q] > red[0] ? red[q] : red[0];
        maxima[(second ? kMaxima : 0) + block] = __builtin_bit_cast(float, red[0]);
    }
}

// The upstream gradient: one number for a reduced loss, one per row for reduction none (these relative to the largest, so that fp16 planes hold
// them).
struct Upstream { const float* g; const float* largest; const float* count; const long long* target; long long ignore; int reduction; float scale; };
// m 2^e, |m| in [1/2, 1) of a number, and the product of such: factors of a gradient may each be far from 1 (a power of two that an operand was scaled
// by, a small upstream gradient), and only what they make of the sums has to fit the type
struct Factor { float m; int e; };
__device__ __forceinline__ Factor factor_of(float v) {
    int e = 0;
    const float m = frexpf(v, &e);
    return fabsf(v) <= 3.4028235e38f ? Factor{m, e} : Factor{v, 0};
}
__device__ __forceinline__ Factor operator*(Factor a, Factor b) { return Factor{a.m * b.m, a.e + b.e}; }
__device__ __forceinline__ f32x4 operator*(f32x4 v, Factor f) { return scaled(v * f.m, f.e); }
__device__ __forceinline__ Factor uniform_factor(const Upstream& u) {
    Factor f = factor_of(u.scale);
    if (u.reduction != 0) f = f * factor_of(u.g[0]);
    if (u.reduction == 1) f.m /= u.count[0];
    return f;
}
__device__ __forceinline__ float row_factor(const Upstream& u, int m) { return u.target[m] == u.ignore ? 0.f : u.reduction == 0 ? u.g[m] : 1.f; }

__global__ __launch_bounds__(1024) void lce_largest_upstream_kernel(Upstream u, int N, float* __restrict__ largest) {
    __shared__ float red[16];
    float top = 0.f;
    for (int i = threadIdx.x; i < N; i += 1024) {
        const float a = fabsf(row_factor(u, i));
        top = a <= 3.4028235e38f ? fmaxf(top, a) : top;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int q = 0; q < 16; ++q) top = fmaxf(top, red[q]);
        largest[0] = top > 0.f ? top : 1.f;
    }
}

// Transposes of a piece of W and (with the first piece) of H, one launch: the first `blocks_w` workgroups take W.  All but fp16, which goes as it
// is: with the exponent of the largest of the `counts` magnitudes that were noted, left in `ex`.  Bound by bytes: 8192 classes of 4096 bf16
// 40 us = 3.4 TB/s.
struct Columns { Source s; u16* dst; long long ldd; int width; const float* maxima; int counts; };
template <class T> constexpr bool kScaled = !__is_same(T, _Float16);
template <class T, int PL>
__global__ __launch_bounds__(256) void pack_transposes_kernel(Columns w, Columns h, int blocks_w, Exponents* __restrict__ ex) {
    __shared__ float red[4];
    const bool second = (int)blockIdx.x >= blocks_w;
    const Columns c = second ? h : w;
    const int id = (int)blockIdx.x - (second ? blocks_w : 0), across = ceil_div(c.width, 64);
    int e = 0;
    if constexpr (kScaled<T>) {
        float m = 0.f;
        for (int i = threadIdx.x; i < c.counts; i += 256) m = fmaxf(m, c.maxima[i]);
        m = wave_largest(m);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
        __syncthreads();
        e = exponent_for(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        if (threadIdx.x == 0 && id == 0) (second ? ex->h : ex->w) = e;
    }
    pack_columns_tile<T, PL, FP16>(c.s, e, c.dst, c.ldd, c.width, id % across, id / across);
}

constexpr int kProbabilityExponent = 14;

// a piece of G and of its transpose: classes [v0, v0 + vp).  G [N][packed vp] holds p - [v = t] (0 where the row is ignored), GT [vp][packed N] the
// same times the row's upstream gradient relative to the largest; columns behind N and vp up to the packed width are zero.  Bound by the matrix
// instructions, and then by its stores: 8192 rows, 8192 classes of 4096 bf16 441 us = 1250 TFLOP/s, 268 MB of it written.
template <class TileT>
__global__ __launch_bounds__(TileT::THREADS, 2) void lce_gradient_kernel(Operand H, Operand W, int width, Logits how,
        const Row* __restrict__ stats, Upstream up, int v0, int vp, int V, u16* __restrict__ G, long long ldg,
        u16* __restrict__ GT, long long ldgt) {
    constexpr int PL = TileT::PL;
    UNFLOW_DYNAMIC_LDS(char, lds);
    const int mt = ceil_div(H.rows, TileT::BM), nt = ceil_div(vp, TileT::BN);
    int tm, tn;
    tile_of(xcd_remap((int)blockIdx.x, (int)gridDim.x), mt, nt, tm, tn);
    const int m0 = tm * TileT::BM, n0 = tn * TileT::BN;
    TileT T;
    const Operand piece{W.p + (long long)v0 * W.ld, W.ld, vp};
    T.run(H, piece, 0, width, m0, n0, lds);
    how.ew += PL == TWO ? v0 : 0;
    const float unit = (float)(1 << kProbabilityExponent);
    const int wide_n = (int)round_up(vp, PL == TWO ? 32 : 8);
    const bool edge = n0 + TileT::BN > vp;
    float weights[TileT::MI];
#pragma unroll
    for (int i = 0; i < TileT::MI; ++i) {
        const int m = m0 + TileT::row(i);
        const bool there = m < H.rows;
        const long long t = there ? up.target[m] : up.ignore, in_tile = t - v0 - n0;
        const bool used = there && t != up.ignore, known = t >= 0 && t < V;
        const Row s = there ? stats[m] : Row{0.f, 0.f, 0.f, 0.f};
        const int own = used && in_tile >= 0 && in_tile < TileT::BN ? (int)in_tile : -1, eh = PL == TWO && there ? how.eh[m] : 0;
        const float inverse = used ? (known ? s.inverse * unit : NAN) : 0.f;
        weights[i] = !used ? 0.f : up.reduction == 0 ? up.g[m] / up.largest[0] : 1.f;
#pragma unroll
        for (int j = 0; j < TileT::NI; ++j) {
            const f32x4 z = logits_of<PL>(how, T.acc[i][j], eh, n0 + TileT::col(j), vp - 1);
            // (z - top is at most 0; the minimum is there for a row that is not used and may hold anything: NaN becomes a number, and 0 times it)
#pragma unroll
            for (int r = 0; r < 4; ++r) T.acc[i][j][r] = exp2_of(fminf(z[r] - s.top, 1.f)) * inverse;
            if (edge)
#pragma unroll
                for (int r = 0; r < 4; ++r) T.acc[i][j][r] = n0 + TileT::col(j) + r < vp ? T.acc[i][j][r] : 0.f;
        }
        if (__ballot(own >= 0))
#pragma unroll
            for (int j = 0; j < TileT::NI; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (TileT::col(j) + r == own) T.acc[i][j][r] = -s.others * unit;
        if (G && there)
#pragma unroll
            for (int j = 0; j < TileT::NI; ++j)
                if (n0 + TileT::col(j) < wide_n) pack4<PL, FP16>(G + (long long)m * ldg, n0 + TileT::col(j), T.acc[i][j]);
    }
    // (a row that is not used, or behind the last, is zeros already: 0 times its weight)
    if (GT) T.template store_transposed<FP16>(lds, GT, ldgt, vp, ldgt, m0, n0, [&](int i, int j) { return T.acc[i][j] * weights[i]; });
}

// The two products of a piece, one launch: job 0 is dH += G W, job 1 dW = G^T H.  C = A B^T in `shares` shares of what is summed.  A job without
// `sums` is one share and goes to the gradient as it is; else the shares' accumulators go to fp32 sums [shares][rows of A][ldc], added to what
// is there unless it is the first piece.  Bound by the matrix instructions: both products of that piece 855 us = 1290 TFLOP/s.
struct Product { Operand A, B; int width, shares, tiles; float* sums; long long ldc; int first; void* out; int by_h; };

// what turns a job's sums into gradients: the uniform factor, and the row's own (dH; for dW it is in GT, relative to the largest)
template <class T> __device__ __forceinline__ Factor product_factor(const Exponents* ex, const Upstream& up, int by_h) {
    Factor f = uniform_factor(up);
    if (by_h && up.reduction == 0) f = f * factor_of(up.largest[0]);
    if constexpr (kScaled<T>) f.e -= by_h ? ex->h : ex->w;
    f.e -= kProbabilityExponent;
    return f;
}

template <class T_, class TileT>
__global__ __launch_bounds__(TileT::THREADS, 2) void lce_products_kernel(Product a, Product b, const Exponents* __restrict__ ex, Upstream up) {
    UNFLOW_DYNAMIC_LDS(char, lds);
    // Each job is dealt over the XCDs by itself: their units differ in length.  (A workgroup that goes through units of its own, as in the forward
    // pass, gains nothing where they are alike and loses a third where they are not.)
    const int units_a = a.tiles * a.shares;
    const bool second = (int)blockIdx.x >= units_a;
    const Product p = second ? b : a;
    const int id = second ? xcd_remap((int)blockIdx.x - units_a, (int)gridDim.x - units_a) : xcd_remap((int)blockIdx.x, units_a);
    const int share = id / p.tiles;
    int tm, tn;
    tile_of(id % p.tiles, ceil_div(p.A.rows, TileT::BM), ceil_div(p.B.rows, TileT::BN), tm, tn);
    const int m0 = tm * TileT::BM, n0 = tn * TileT::BN;
    const int per = ceil_div(ceil_div(p.width, 64), p.shares) * 64;
    const int k0 = share * per, k1 = k0 + per < p.width ? k0 + per : p.width;
    TileT T;
    T.run(p.A, p.B, k0, k1, m0, n0, lds);
    if (p.sums) {
        float* C = p.sums + (long long)share * p.A.rows * p.ldc;
#pragma unroll
        for (int i = 0; i < TileT::MI; ++i) {
            const int m = m0 + TileT::row(i);
            if (m >= p.A.rows) continue;
            float* row = C + (long long)m * p.ldc;
            if (!p.first) {                                            // (all of a row's loads before its sums: one wait, not one per load)
                f32x4 old[TileT::NI];
#pragma unroll
                for (int j = 0; j < TileT::NI; ++j) {
                    const int n = n0 + TileT::col(j);
                    old[j] = n < p.ldc ? *reinterpret_cast<const f32x4*>(row + n) : f32x4{0.f, 0.f, 0.f, 0.f};
                }
#pragma unroll
                for (int j = 0; j < TileT::NI; ++j) T.acc[i][j] += old[j];
            }
#pragma unroll
            for (int j = 0; j < TileT::NI; ++j)
                // (ldc: the columns rounded up to 4)
                if (n0 + TileT::col(j) < p.ldc) *reinterpret_cast<f32x4*>(row + n0 + TileT::col(j)) = T.acc[i][j];
        }
        return;
    }
    const Factor f = product_factor<T_>(ex, up, p.by_h);
#pragma unroll
    for (int i = 0; i < TileT::MI; ++i) {
        const int m = m0 + TileT::row(i);
        if (m >= p.A.rows) continue;
        const Factor fm = p.by_h ? f : f * factor_of(row_factor(up, m));
#pragma unroll
        for (int j = 0; j < TileT::NI; ++j) {
            const int n = n0 + TileT::col(j), left = p.B.rows - n;
            if (left > 0) store4<T_>((T_*)p.out + (long long)m * p.B.rows + n, T.acc[i][j] * fm, left < 4 ? left : 4);
        }
    }
}

// gradients = sums over the shares, in order, times the factors; one launch for the jobs that have sums (blocks of the first, then of the second).
// Bound by bytes: 4096 x 2048 to bf16 11 us = 4.5 TB/s.
template <class T_>
__global__ __launch_bounds__(256) void lce_finish_kernel(Product a, Product b, int blocks_a, const Exponents* __restrict__ ex, Upstream up) {
    const bool second = (int)blockIdx.x >= blocks_a;
    const Product p = second ? b : a;
    const int block = (int)blockIdx.x - (second ? blocks_a : 0), blocks = second ? (int)gridDim.x - blocks_a : blocks_a;
    const Factor f = product_factor<T_>(ex, up, p.by_h);
    const int rows = p.A.rows, cols = p.B.rows;
    const long long per = p.ldc / 4, total = per * rows;
    for (long long g = block * 256ll + threadIdx.x; g < total; g += blocks * 256ll) {
        const long long r = g / per;
        const int n = (int)(g - r * per) * 4;
        f32x4 v = *reinterpret_cast<const f32x4*>(p.sums + r * p.ldc + n);
        for (int s = 1; s < p.shares; ++s) v += *reinterpret_cast<const f32x4*>(p.sums + ((long long)s * rows + r) * p.ldc + n);
        store4<T_>((T_*)p.out + r * cols + n, v * (p.by_h ? f : f * factor_of(row_factor(up, (int)r))), cols - n < 4 ? cols - n : 4);
    }
}

// ---- the host side
#define LAUNCH_TILES(kernel, count, lds, ...)                                                                                  \
    do {                                                                                                                       \
        if (lds > 65536) (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);      \
        UNFLOW_LAUNCH(kernel, dim3(count), dim3(TileT::THREADS), lds, stream, __VA_ARGS__);                                    \
    } while (0)
// workgroups of a kernel that goes through its tiles itself
template <class TileT> static int resident(long long units) { return (int)(units < 256 * TileT::PER_CU ? units : 256 * TileT::PER_CU); }
template <int PL, int EL, class F> static void with_tile(int size, F&& f) {
    if (size == 0) f(Tile<256, 256, 2, 4, 2, PL, EL>{});
    else if (size == 1) f(Tile<192, 192, 2, 4, 3, PL, EL>{});
    else if (size == 2) f(Tile<128, 128, 2, 2, 2, PL, EL>{});
    else if (size == 3) f(Tile<64, 64, 2, 2, 2, PL, EL>{});
    else if (size == 4) f(Tile<128, 128, 2, 2, 4, PL, EL>{});
    else f(Tile<64, 64, 2, 2, 4, PL, EL>{});
}

// the packed inputs of a call, as bits
enum { kPackedH = 1, kPackedW = 2, kPackedBoth = 3 };

// What a call needs of its buffers, and where.  `kept` is what the forward pass leaves for the backward pass: statistics of the rows, and those of the
// inputs that it has packed (`held`).  Where the backward pass finds an input neither held nor fit to be read in place, it packs it into its
// workspace: the two passes may see the same inputs in different layouts.
struct Layout { long long maxima, eh, ew, hp, wp; };     // of packed inputs (offsets; those of what is not there are not used)
struct Plan {
    int planes;
    bool few;
    int packed, held;
    long long wd, wn;                    // packed widths of D and N
    long long stats, kept_bytes;
    Layout in_kept, in_workspace;
    int size_z;
    long long partial, ztarget, losses, forward_bytes;
    int vp, size_g, size_p, limit;
    long long wvp, ldc;
    long long magnitudes, exponents, largest, g, gt, ht, wt, sum_h, sum_w, backward_bytes;
};

// classes a workgroup of lce_few_kernel takes
static int few_classes(int N) { return N <= 16 ? 64 : 32; }

// 16-byte loads of whole rows
static bool aligned(const void* p, long long ld, int D, int dtype) {
    const int each = dtype == kFp32 ? 4 : 8;
    return D % each == 0 && ld % each == 0 && ((size_t)p & 15) == 0;
}

struct Taken {
    long long bytes = 0;
    long long operator()(long long n) { const long long at = bytes; bytes += round_up(n, 256); return at; }
};
static Layout layout_of(Taken& take, int packed, int planes, int N, int V, long long wd) {
    Layout l{};
    if (packed && planes == TWO) {
        l.maxima = take(2 * kMaxima * 4);
        l.eh = take(4ll * N);
        l.ew = take(4ll * V);
    }
    if (packed & kPackedH) l.hp = take(2 * wd * N);
    if (packed & kPackedW) l.wp = take(2 * wd * V);
    return l;
}
// The size of what is kept also says what it holds: whole lines of 256 bytes, and the bits of the packed inputs.  Two layouts never have one size.
static long long kept_of(Plan& p, int N, int V) {
    Taken take;
    p.stats = take(4ll * (4 * (long long)N + 1));
    p.in_kept = layout_of(take, p.held, p.planes, N, V, p.wd);
    return take.bytes + p.held;
}

// held: the inputs that `kept` holds packed, of a backward pass; -1: a forward pass decides that
static Plan plan_of(const void* h, long long ldh, const void* w, long long ldw, int N, int V, int D, int dtype, int held, bool train, bool need_h,
        bool need_w) {
    Plan p{};
    p.planes = dtype == kFp32 ? TWO : ONE;
    p.wd = packed_width(p.planes, D);
    p.wn = packed_width(p.planes, N);
    p.packed = dtype == kFp32 ? kPackedBoth : (aligned(h, ldh, D, dtype) ? 0 : kPackedH) | (aligned(w, ldw, D, dtype) ? 0 : kPackedW);
    p.few = N <= (dtype == kFp32 ? 64 : p.packed & kPackedW ? 32 : 16) && D >= (dtype == kFp32 ? 4 : 8);
    p.held = held >= 0 ? held : p.few ? 0 : p.packed;
    p.packed |= p.held;
    p.kept_bytes = kept_of(p, N, V);
    long long at = 0;
    auto take = [&](long long bytes) { const long long a = at; at += round_up(bytes, 256); return a; };
    const Job z{N, V, stages_of(p.wd), false, false, 0.};
    p.size_z = choose(p.planes, &z, 1).size;
    p.partial = take(8ll * ceil_div(V, p.few ? few_classes(N) : kSizes[p.size_z]) * N);
    p.ztarget = take(4ll * N);
    p.losses = take(4ll * N);
    p.forward_bytes = at;
    if (!train) return p;
    Taken repacked;
    p.in_workspace = layout_of(repacked, p.packed & ~p.held, p.planes, N, V, p.wd);
    at = repacked.bytes;
    // A piece of G and its transpose take 256 MB at most (and hold 1024 classes at least): as long as a piece's two products fill the chip and
    // sum over thousands of classes, larger pieces gain nothing.
    const long long per_class = 2ll * p.planes * 2 * round_up(N, 32);
    long long vp = (256ll << 20) / per_class;
    vp = vp < 1024 ? 1024 : vp / 256 * 256;
    if (vp > 65536) vp = 65536;
    const long long pieces = (V + vp - 1) / vp;
    vp = round_up((V + pieces - 1) / pieces, 256);                       // equal pieces
    p.vp = (int)(vp < V ? vp : V);
    p.wvp = packed_width(p.planes, p.vp);
    const Job g{N, p.vp, stages_of(p.wd), false, false, 4. * p.planes};
    p.size_g = choose(p.planes, &g, 1).size;
    Job both[2];
    int jobs = 0;
    if (need_h) both[jobs++] = Job{N, D, stages_of(p.wvp), false, true, p.vp < V ? 8. : 2. * p.planes};
    if (need_w) both[jobs++] = Job{p.vp, D, stages_of(p.wn), false, true, 2. * p.planes};
    if (jobs) {
        const Choice c = choose(p.planes, both, jobs);
        p.size_p = c.size;
        p.limit = c.limit;
    }
    if (dtype == kBf16) p.magnitudes = take(2 * kMaxima * 4);
    p.exponents = take(sizeof(Exponents));
    p.largest = take(4);
    p.g = take(2 * p.wvp * N);
    p.gt = take(2 * p.wn * p.vp);
    p.ldc = round_up(D, 4);
    if (need_h) {
        p.wt = take(2 * p.wvp * D);
        p.sum_h = take(4ll * shares_of(stages_of(p.wvp), p.limit) * p.ldc * N);
    }
    if (need_w) {
        p.ht = take(2 * p.wn * D);
        const int shares = shares_of(stages_of(p.wn), p.limit);
        if (shares > 1) p.sum_w = take(4ll * shares * p.ldc * p.vp);
    }
    p.backward_bytes = at;
    return p;
}

static int blocks_for(long long work) { const long long b = (work + 255) / 256; return (int)(b < 1 ? 1 : b > 4096 ? 4096 : b); }

struct Inputs { const void* h; long long ldh; const void* w; long long ldw; const long long* target; long long ignore; int N, V, D; float scale; };

static int pack_blocks(int rows) { return rows > 4 * kMaxima ? kMaxima : ceil_div(rows, 4); }

// H and W as operands: as they are, packed in `kept` or packed in `ws`; those of `pack` are packed now (where they go: all of them in one buffer).
// The largest magnitudes of packed fp32 inputs are left in `maxima`.
template <class T, int PL, int EL>
static Logits operands(const Plan& p, const Inputs& in, int pack, char* kept, char* ws, hipStream_t stream, Operand& H, Operand& W,
        float*& maxima) {
    u16 *hp = (u16*)(p.held & kPackedH ? kept + p.in_kept.hp : ws + p.in_workspace.hp),
        *wp = (u16*)(p.held & kPackedW ? kept + p.in_kept.wp : ws + p.in_workspace.wp);
    // (fp32 inputs are packed both or not at all, into one buffer)
    const Layout& l = p.held ? p.in_kept : p.in_workspace;
    char* of_both = p.held ? kept : ws;
    H = p.packed & kPackedH ? Operand{hp, p.wd, in.N} : Operand{(const u16*)in.h, in.ldh, in.N};
    W = p.packed & kPackedW ? Operand{wp, p.wd, in.V} : Operand{(const u16*)in.w, in.ldw, in.V};
    maxima = (float*)(of_both + l.maxima);
    const Packed at{hp, wp, (int*)(of_both + l.eh), (int*)(of_both + l.ew), maxima};
    if (pack) {
        const int blocks_h = pack & kPackedH ? pack_blocks(in.N) : 0, blocks_w = pack & kPackedW ? pack_blocks(in.V) : 0;
        UNFLOW_LAUNCH((pack_inputs_kernel<T, PL, EL>), dim3(blocks_h + blocks_w), dim3(256), 0, stream,
            Source{in.h, in.ldh, in.N, in.D, in.target, in.ignore}, Source{in.w, in.ldw, in.V, in.D}, blocks_h, at, p.wd,
            (int)(PL == TWO ? p.wd / 2 : p.wd));
    }
    return Logits{in.scale * kLog2E, at.eh, at.ew};
}

template <class T, int PL, int EL>
static void forward(const Plan& p, const Inputs& in, int reduction, float* loss, char* kept, char* ws, hipStream_t stream) {
    float* stats = (float*)(kept + p.stats);
    float2* partial = (float2*)(ws + p.partial);
    float* zt = (float*)(ws + p.ztarget);
    float* losses = reduction == 0 ? loss : (float*)(ws + p.losses);
    int columns;
    if (p.few) {
        columns = ceil_div(in.V, few_classes(in.N));
        auto launch = [&](auto kernel) {
            UNFLOW_LAUNCH(kernel, dim3(columns), dim3(256), 0, stream, (const T*)in.h, in.ldh, (const T*)in.w, in.ldw, in.N, in.V, in.D,
                in.scale * kLog2E, in.target, partial, zt);
        };
        if (in.N <= 16) launch(lce_few_kernel<T, 1, 4, 4>);
        // (beyond 16 rows a wave holds fewer classes and steps, so that more waves fit a CU)
        else if (in.N <= 32) launch(lce_few_kernel<T, 2, 2, 4>);
        else if constexpr (PL == TWO) launch(lce_few_kernel<T, 4, 2, 2>);
    } else {
        Operand H, W;
        float* maxima;
        const Logits how = operands<T, PL, EL>(p, in, p.packed, kept, ws, stream, H, W, maxima);
        columns = ceil_div(in.V, kSizes[p.size_z]);
        with_tile<PL, EL>(p.size_z, [&](auto tile) {
            using TileT = decltype(tile);
            LAUNCH_TILES((lce_forward_kernel<TileT>), resident<TileT>(tiles_of(in.N, in.V, TileT::BM)),
                TileT::STAGES_LDS + TileT::WN * TileT::BM * (int)sizeof(float2), H, W, (int)p.wd, how, in.target, partial, zt);
        });
    }
    const float2* pairs = partial;
    const float* own = zt;
    Row* rows = (Row*)stats;
    float* count = stats + 4ll * in.N;
    if (reduction != 0 && in.N <= 1024 && columns <= 32) {
        UNFLOW_LAUNCH(lce_join_reduce_kernel, dim3(1), dim3(1024), 0, stream, pairs, columns, in.N, in.V, in.target, in.ignore, own, rows,
            reduction == 1 ? 1 : 0, loss, count);
        return;
    }
    // (a workgroup for 16 rows reads their pairs in whole lines; few rows over many columns need more of them)
    if (in.N <= 256) UNFLOW_LAUNCH((lce_join_kernel<1>), dim3(in.N), dim3(256), 0, stream, pairs, columns, in.N, in.V, in.target, in.ignore, own,
        rows, losses);
    else UNFLOW_LAUNCH((lce_join_kernel<16>), dim3(ceil_div(in.N, 16)), dim3(256), 0, stream, pairs, columns, in.N, in.V, in.target, in.ignore, own,
        rows, losses);
    if (reduction != 0) UNFLOW_LAUNCH(lce_reduce_kernel, dim3(1), dim3(1024), 0, stream, (const float*)losses, in.target, in.ignore, in.N,
        reduction == 1 ? 1 : 0, loss, count);
}

template <class T, int PL, int EL>
static void backward(const Plan& p, const Inputs& in, int reduction, const float* gout, void* dh, void* dw, char* kept, char* ws,
        hipStream_t stream) {
    const float* stats = (const float*)(kept + p.stats);
    Operand H, W;
    float* maxima;
    const Logits how = operands<T, PL, EL>(p, in, p.packed & ~p.held, kept, ws, stream, H, W, maxima);
    Exponents* ex = (Exponents*)(ws + p.exponents);
    if (PL == ONE) maxima = (float*)(ws + p.magnitudes);
    if constexpr (kScaled<T> && PL == ONE) {
        const int blocks_h = dw ? pack_blocks(in.N) : 0, blocks_w = dh ? pack_blocks(in.V) : 0;
        UNFLOW_LAUNCH(lce_magnitudes_kernel, dim3(blocks_h + blocks_w), dim3(256), 0, stream, H, W, (int)(p.wd / 8), blocks_h, in.target, in.ignore,
            maxima);
    }
    const Upstream up{gout, (const float*)(ws + p.largest), stats + 4ll * in.N, in.target, in.ignore, reduction, in.scale};
    if (reduction == 0) UNFLOW_LAUNCH(lce_largest_upstream_kernel, dim3(1), dim3(1024), 0, stream, up, in.N, (float*)(ws + p.largest));
    u16 *G = (u16*)(ws + p.g), *GT = (u16*)(ws + p.gt);
    const bool single = p.vp >= in.V;
    for (int v0 = 0; v0 < in.V; v0 += p.vp) {
        const int vp = in.V - v0 < p.vp ? in.V - v0 : p.vp;
        const long long wvp = packed_width(PL, vp);
        Columns wc{}, hc{};
        int blocks_w = 0, blocks_h = 0;
        if (dh) {
            wc = Columns{Source{(const T*)in.w + (long long)v0 * in.ldw, in.ldw, vp, in.D}, (u16*)(ws + p.wt), wvp,
                (int)(PL == TWO ? wvp / 2 : wvp), maxima + kMaxima, pack_blocks(in.V)};
            blocks_w = ceil_div(wc.width, 64) * ceil_div(in.D, 64);
        }
        if (dw && v0 == 0) {
            hc = Columns{Source{in.h, in.ldh, in.N, in.D, in.target, in.ignore}, (u16*)(ws + p.ht), p.wn, (int)(PL == TWO ? p.wn / 2 : p.wn),
                maxima, pack_blocks(in.N)};
            blocks_h = ceil_div(hc.width, 64) * ceil_div(in.D, 64);
        }
        if (blocks_w + blocks_h) UNFLOW_LAUNCH((pack_transposes_kernel<T, PL>), dim3(blocks_w + blocks_h), dim3(256), 0, stream, wc, hc,
            blocks_w, ex);
        with_tile<PL, EL>(p.size_g, [&](auto tile) {
            using TileT = decltype(tile);
            LAUNCH_TILES((lce_gradient_kernel<TileT>), (int)tiles_of(in.N, vp, TileT::BM), TileT::LDS, H, W, (int)p.wd, how, (const Row*)stats, up,
                v0, vp, in.V, dh ? G : nullptr, p.wvp, dw ? GT : nullptr, p.wn);
        });
        Product a{}, b{};
        a.shares = b.shares = 1;
        if (dh) {
            a = Product{Operand{G, p.wvp, in.N}, Operand{(const u16*)(ws + p.wt), wvp, in.D}, (int)wvp, shares_of(stages_of(p.wvp), p.limit), 0,
                (float*)(ws + p.sum_h), p.ldc, v0 == 0 ? 1 : 0, dh, 0};
            if (single && a.shares == 1) a.sums = nullptr;
        }
        if (dw) {
            b = Product{Operand{GT, p.wn, vp}, Operand{(const u16*)(ws + p.ht), p.wn, in.D}, (int)p.wn, shares_of(stages_of(p.wn), p.limit), 0,
                (float*)(ws + p.sum_w), p.ldc, 1, (T*)dw + (long long)v0 * in.D, 1};
            if (b.shares == 1) b.sums = nullptr;
        }
        with_tile<PL, FP16>(p.size_p, [&](auto tile) {
            using TileT = decltype(tile);
            if (dh) a.tiles = (int)tiles_of(in.N, in.D, TileT::BM);
            if (dw) b.tiles = (int)tiles_of(vp, in.D, TileT::BM);
            const bool swap = dw && (!dh || b.width / b.shares > a.width / a.shares);        // the longer units first
            LAUNCH_TILES((lce_products_kernel<T, TileT>), a.tiles * a.shares + b.tiles * b.shares, TileT::STAGES_LDS, swap ? b : a, swap ? a : b,
                (const Exponents*)ex, up);
        });
        const bool last = v0 + vp >= in.V;
        const int finish_a = dh && last && a.sums ? blocks_for((long long)in.N * (p.ldc / 4)) : 0,
            finish_b = dw && b.sums ? blocks_for((long long)vp * (p.ldc / 4)) : 0;
        if (finish_a + finish_b) UNFLOW_LAUNCH((lce_finish_kernel<T>), dim3(finish_a + finish_b), dim3(256), 0, stream, a, b, finish_a,
            (const Exponents*)ex, up);
    }
}

static bool sizes_ok(long long ldh, long long ldw, int N, int V, int D, int dtype, int reduction) {
    return N > 0 && V > 0 && D > 0 && N <= UNFLOW_LCE_MAX_ROWS && V <= UNFLOW_LCE_MAX_CLASSES && D <= UNFLOW_LCE_MAX_DIM &&
           ldh >= D && ldw >= D && ldh <= UNFLOW_LCE_MAX_DIM && ldw <= UNFLOW_LCE_MAX_DIM &&
           dtype >= kFp32 && dtype <= kFp16 && reduction >= 0 && reduction <= 2;
}

}  // namespace

extern "C" int unflow_linear_ce_workspace(const void* hidden, long long ldh, const void* weight, long long ldw, int N, int V, int D, int dtype,
        int need_dhidden, int need_dweight, long long* kept_bytes, long long* forward_bytes, long long* backward_bytes) {
    UNFLOW_REQUIRE(kept_bytes && forward_bytes && backward_bytes && sizes_ok(ldh, ldw, N, V, D, dtype, 0));
    const Plan p = plan_of(hidden, ldh, weight, ldw, N, V, D, dtype, -1, need_dhidden || need_dweight, need_dhidden != 0, need_dweight != 0);
    *kept_bytes = p.kept_bytes;
    *forward_bytes = p.forward_bytes;
    *backward_bytes = p.backward_bytes;
    return 0;
}

// what a buffer of this size holds, or -1 where no forward pass of these sizes keeps as much
static int held_in(long long kept_bytes, int N, int V, int D, int dtype) {
    if (kept_bytes < 0) return -1;
    Plan p{};
    p.planes = dtype == kFp32 ? TWO : ONE;
    p.wd = packed_width(p.planes, D);
    p.held = (int)(kept_bytes % 256);
    if (p.held > kPackedBoth || (dtype == kFp32 && p.held != 0 && p.held != kPackedBoth) || kept_of(p, N, V) != kept_bytes) return -1;
    return p.held;
}

extern "C" int unflow_linear_ce_bwd_workspace(const void* hidden, long long ldh, const void* weight, long long ldw, int N, int V, int D, int dtype,
        int need_dhidden, int need_dweight, long long kept_bytes, long long* backward_bytes) {
    UNFLOW_REQUIRE(backward_bytes && (need_dhidden || need_dweight) && sizes_ok(ldh, ldw, N, V, D, dtype, 0));
    const int held = held_in(kept_bytes, N, V, D, dtype);
    UNFLOW_REQUIRE(held >= 0);
    *backward_bytes = plan_of(hidden, ldh, weight, ldw, N, V, D, dtype, held, true, need_dhidden != 0, need_dweight != 0).backward_bytes;
    return 0;
}

// kept_bytes -1: as large as unflow_linear_ce_workspace said, by the caller's word
static int forward_call(const void* hidden, long long ldh, const void* weight, long long ldw, const long long* target, int N, int V, int D, int dtype,
        float scale, long long ignore_index, int reduction, float* loss, void* kept, long long kept_bytes, void* workspace,
        long long workspace_bytes, void* stream) {
    UNFLOW_REQUIRE(hidden && weight && target && loss && kept && workspace && sizes_ok(ldh, ldw, N, V, D, dtype, reduction));
    UNFLOW_REQUIRE(((size_t)kept & 15) == 0 && ((size_t)workspace & 15) == 0);
    const Plan p = plan_of(hidden, ldh, weight, ldw, N, V, D, dtype, -1, false, false, false);
    UNFLOW_REQUIRE(workspace_bytes >= p.forward_bytes && (kept_bytes == -1 || kept_bytes == p.kept_bytes));
    const Inputs in{hidden, ldh, weight, ldw, target, ignore_index, N, V, D, scale};
    char *k = (char*)kept, *ws = (char*)workspace;
    if (dtype == kFp32) forward<float, TWO, FP16>(p, in, reduction, loss, k, ws, (hipStream_t)stream);
    else if (dtype == kBf16) forward<__bf16, ONE, BF16>(p, in, reduction, loss, k, ws, (hipStream_t)stream);
    else forward<_Float16, ONE, FP16>(p, in, reduction, loss, k, ws, (hipStream_t)stream);
    return unflow_launch_status();
}

extern "C" int unflow_linear_ce_fwd(const void* hidden, long long ldh, const void* weight, long long ldw, const long long* target, int N, int V,
        int D, int dtype, float scale, long long ignore_index, int reduction, float* loss, void* kept, void* workspace, long long workspace_bytes,
        void* stream) {
    return forward_call(hidden, ldh, weight, ldw, target, N, V, D, dtype, scale, ignore_index, reduction, loss, kept, -1, workspace, workspace_bytes,
        stream);
}

extern "C" int unflow_linear_ce_fwd_ex(const void* hidden, long long ldh, const void* weight, long long ldw, const long long* target, int N, int V,
        int D, int dtype, float scale, long long ignore_index, int reduction, float* loss, void* kept, long long kept_bytes, void* workspace,
        long long workspace_bytes, void* stream) {
    UNFLOW_REQUIRE(kept_bytes >= 0);
    return forward_call(hidden, ldh, weight, ldw, target, N, V, D, dtype, scale, ignore_index, reduction, loss, kept, kept_bytes, workspace,
        workspace_bytes, stream);
}

// held -1: what a forward pass over these very pointers keeps
static int backward_call(const void* hidden, long long ldh, const void* weight, long long ldw, const long long* target, const float* gout, int N, int V,
        int D, int dtype, float scale, long long ignore_index, int reduction, void* dhidden, void* dweight, const void* kept, int held,
        void* workspace, long long workspace_bytes, void* stream) {
    UNFLOW_REQUIRE(hidden && weight && target && gout && (dhidden || dweight) && kept && workspace && sizes_ok(ldh, ldw, N, V, D, dtype, reduction));
    UNFLOW_REQUIRE(((size_t)kept & 15) == 0 && ((size_t)workspace & 15) == 0);
    const Plan p = plan_of(hidden, ldh, weight, ldw, N, V, D, dtype, held, true, dhidden != nullptr, dweight != nullptr);
    UNFLOW_REQUIRE(workspace_bytes >= p.backward_bytes);
    const Inputs in{hidden, ldh, weight, ldw, target, ignore_index, N, V, D, scale};
    char *k = (char*)const_cast<void*>(kept), *ws = (char*)workspace;
    if (dtype == kFp32) backward<float, TWO, FP16>(p, in, reduction, gout, dhidden, dweight, k, ws, (hipStream_t)stream);
    else if (dtype == kBf16) backward<__bf16, ONE, BF16>(p, in, reduction, gout, dhidden, dweight, k, ws, (hipStream_t)stream);
    else backward<_Float16, ONE, FP16>(p, in, reduction, gout, dhidden, dweight, k, ws, (hipStream_t)stream);
    return unflow_launch_status();
}

extern "C" int unflow_linear_ce_bwd(const void* hidden, long long ldh, const void* weight, long long ldw, const long long* target,
        const float* gout, int N, int V, int D, int dtype, float scale, long long ignore_index, int reduction, void* dhidden, void* dweight,
        const void* kept, void* workspace, long long workspace_bytes, void* stream) {
    return backward_call(hidden, ldh, weight, ldw, target, gout, N, V, D, dtype, scale, ignore_index, reduction, dhidden, dweight, kept, -1, workspace,
        workspace_bytes, stream);
}

extern "C" int unflow_linear_ce_bwd_ex(const void* hidden, long long ldh, const void* weight, long long ldw, const long long* target,
        const float* gout, int N, int V, int D, int dtype, float scale, long long ignore_index, int reduction, void* dhidden, void* dweight,
        const void* kept, long long kept_bytes, void* workspace, long long workspace_bytes, void* stream) {
    UNFLOW_REQUIRE(sizes_ok(ldh, ldw, N, V, D, dtype, reduction));
    const int held = held_in(kept_bytes, N, V, D, dtype);
    UNFLOW_REQUIRE(held >= 0);
    return backward_call(hidden, ldh, weight, ldw, target, gout, N, V, D, dtype, scale, ignore_index, reduction, dhidden, dweight, kept, held, workspace,
        workspace_bytes, stream);
}
