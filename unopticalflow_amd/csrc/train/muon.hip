// Orthogonalisation by Newton-Schulz products, and the optimiser step made of it (Muon), over a list of matrices of any shapes at once.
//
//   X_0 = G / (|G|_F + eps)          (G^T where G has more rows than columns: m <= n from here on)
//   S = X X^T,  Q = a I + b S + c S S,  X <- Q X,       `steps` times
//   step: M += (1 - mu)(G - M),  U = G + mu (M - G) (nesterov) or M,  P = P (1 - lr wd) - lr sqrt(max(1, rows / cols)) X(U)
//
// S and Q are symmetric: their tiles above the diagonal are not computed but written as the mirror of those below, so a step costs
// m^2 n + m^3 + 2 m^2 n operations instead of 4 m^2 n + 2 m^3.  The products bound large matrices; a list of small ones is bound by launches,
// so every phase is one launch over the tiles of all matrices (a wave finds its matrix in a table of running tile counts), 3 launches a step, 4
// where S is summed in shares.
// Matrices of up to 32 rows or columns, where nothing larger is in the list, have kernels of their own (in the middle of this file).
//
// Numbers of the tiles (mfma16.h): every type is iterated on as two fp16 planes (22 bits, products and sums as in fp32).  One plane would
// take a third of the products, and its 2^-12 looks small beside the 2^-9 of a bf16 result, but the iteration multiplies small singular values by
// a^5 = 485 and what rounding spreads over their directions with them: a bf16 matrix of low rank comes out several percent off that way.  The
// Frobenius norm is summed in 64 bits.  |X|, |S|, |Q| are bounded by the polynomial over [0, 1], which gives the powers of two that
// the planes are scaled by.  A matrix whose norm is far below eps comes out as nearly zero, as the definition has it, but without relative
// accuracy.
#include "pack.h"
#include "plan.h"
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>

namespace {

constexpr int kFp32 = 0, kBf16 = 1, kFp16 = 2;                     // UNFLOW_DTYPE_*

struct Problem {
    const void* x;               // gradient / input
    void* out;                   // parameter / output
    float* momentum;
    long long X, XT0, XT1, S, Q; // byte offsets into the workspace
    long long shares_at;         // byte offset of the partial sums of S
    int rows, cols, m, n;
    int part0, parts;            // its sums of squares
    int shares;                  // S is summed over n in this many parts
    float boost;                 // sqrt(max(1, rows / cols))
};
static_assert(sizeof(Problem) % 4 == 0, "copied by words");

// running counts of the work items of all problems, one row per phase
enum { kNorm, kPack, kSquare, kJoin, kPoly, kApply, kPhases };
// behind them, for the three product phases: first and last + 1 work item of the matrices of the same length
enum { kSquareClass = kPhases, kPolyClass = kSquareClass + 2, kApplyClass = kPolyClass + 2, kTables = kApplyClass + 2 };

struct Exponents { int x, s, q; };                                 // planes hold X 2^x, S 2^s, Q 2^q

// host structures into the workspace through kernel arguments: nothing is copied by the runtime, so a captured call holds no host memory
constexpr int kPiece = 896;
struct Words { unsigned w[kPiece]; };
__global__ __launch_bounds__(256) void write_table_kernel(Words src, int count, unsigned* __restrict__ dst) {
    for (int i = threadIdx.x; i < count; i += 256) dst[i] = src.w[i];
}

// How many of the first `count` running counts are at most id.
__device__ __forceinline__ int counts_until(const int* __restrict__ ends, int count, int id) {
    int at = 0;
    for (int base = 0; base < count; base += 64) {
        const int lane = base + ((int)threadIdx.x & 63), before = __popcll(__ballot((lane < count ? ends[lane] : 0x7fffffff) <= id));
        at += before;
        if (before < 64) break;
    }
    return __builtin_amdgcn_readfirstlane(at);
}
// the problem that work item `id` of a phase belongs to, and the item's number within it
__device__ __forceinline__ int problem_of(const int* __restrict__ ends, int count, int id, int& local) {
    const int at = counts_until(ends, count, id);
    local = id - (at > 0 ? ends[at - 1] : 0);
    return at;
}
// The same for the product phases.  Work items are sorted by length, the longest first; the matrices of one length are dealt over the XCDs by
// themselves, so that every XCD has its share of the long ones and a matrix stays in one L2 as far as it goes.  Up to 64 matrices every lane holds
// one's counts and the search waits for memory once (a launch over small matrices is all latency: 0.5 us for every load that waits for another).
__device__ __forceinline__ int dealt_problem_of(const int* __restrict__ ends, int count, const int* __restrict__ classes, int& local) {
    if (count <= 64) {
        const int lane = (int)threadIdx.x & 63, mine = lane < count ? lane : count - 1;
        const int e = lane < count ? ends[mine] : 0x7fffffff, first = classes[2 * mine], end = classes[2 * mine + 1];
        const int at = __builtin_amdgcn_readfirstlane(__popcll(__ballot(e <= (int)blockIdx.x)));
        const int f = __builtin_amdgcn_readlane(first, at), id = f + xcd_remap((int)blockIdx.x - f, __builtin_amdgcn_readlane(end, at) - f);
        const int owner = __builtin_amdgcn_readfirstlane(__popcll(__ballot(e <= id)));
        const int before = __builtin_amdgcn_readlane(e, owner > 0 ? owner - 1 : 0);
        local = id - (owner > 0 ? before : 0);
        return owner;
    }
    const int at = counts_until(ends, count, (int)blockIdx.x), first = classes[2 * at], end = classes[2 * at + 1];
    return problem_of(ends, count, first + xcd_remap((int)blockIdx.x - first, end - first), local);
}

__device__ __forceinline__ float direction(float g, float m, float mu, int nesterov) { return nesterov ? g + mu * (m - g) : m; }

// ---- sum of squares of a chunk of `size` numbers (after the momentum's update).  Bound by bytes: 16 bf16 weights
// of 1024 x 1024, four of 4096 x 1024 and four of 1024 x 4096 (50 million numbers) with their momenta 91 us = 5.5 TB/s
template <class T, bool STEP>
__global__ __launch_bounds__(256) void norm_kernel(const Problem* __restrict__ table, const int* __restrict__ ends, int count, int size, float mu,
        int nesterov, double* __restrict__ parts) {
    int chunk;
    const Problem p = table[problem_of(ends, count, (int)blockIdx.x, chunk)];
    const long long total = (long long)p.rows * p.cols, e0 = (long long)chunk * size;
    const T* x = (const T*)p.x;
    double sum = 0.;
    for (int k = 0; k < size / 1024; ++k) {
        const long long e = e0 + k * 1024 + threadIdx.x * 4;
        const long long left = total - e;
        if (left <= 0) break;
        const int n = left < 4 ? (int)left : 4;
        f32x4 v = load4(x + e, n);
        if constexpr (STEP) {
            f32x4 m = load4(p.momentum + e, n);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                m[r] = m[r] + (1.f - mu) * (v[r] - m[r]);
                v[r] = direction(v[r], m[r], mu, nesterov);
            }
            store4<float>(p.momentum + e, m, n);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (r >= n) v[r] = 0.f;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += (double)v[r] * (double)v[r];
    }
    __shared__ double red[256];
    red[threadIdx.x] = sum;
    __syncthreads();
#pragma unroll
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) parts[p.part0 + chunk] = red[0];
}

// ---- X_0 and its transpose, as planes: a 64 x 64 tile of the matrix per workgroup, both ways.  Bound by bytes: the same weights 148 us = 4.8 TB/s
template <class T, bool STEP>
__global__ __launch_bounds__(256) void start_kernel(const Problem* __restrict__ table, const int* __restrict__ ends, int count,
        const double* __restrict__ parts, float mu, int nesterov, float eps,
        Exponents ex, char* __restrict__ ws) {
    __shared__ float tile[64][65];
    __shared__ double red[256];
    int id;
    const Problem p = table[problem_of(ends, count, (int)blockIdx.x, id)];
    double sum = 0.;
    for (int i = threadIdx.x; i < p.parts; i += 256) sum += parts[p.part0 + i];
    red[threadIdx.x] = sum;
    __syncthreads();
#pragma unroll
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    // 2^x / (norm + eps), in two factors: the norm may be far from 1 (the division in 64 bits keeps matrices of huge or tiny numbers exact)
    const double factor = ldexp(1.0 / (sqrt(red[0]) + (double)eps), ex.x);
    const int across = ceil_div(p.cols, 64), r0 = id / across * 64, c0 = id % across * 64;
    const bool wide = p.rows <= p.cols;
    u16* straight = (u16*)(ws + (wide ? p.X : p.XT0));               // [rows][packed cols]
    u16* turned = (u16*)(ws + (wide ? p.XT0 : p.X));                 // [cols][packed rows]
    const long long lds_ = packed_width(TWO, p.cols), ldt = packed_width(TWO, p.rows);
    const int wide_c = (int)(lds_ / 2), wide_r = (int)(ldt / 2);
    const int x = (threadIdx.x & 15) * 4, y = threadIdx.x >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = r0 + y + 16 * i, c = c0 + x;
        f32x4 v{0.f, 0.f, 0.f, 0.f};
        if (r < p.rows && c < p.cols) {
            const int n = p.cols - c < 4 ? p.cols - c : 4;
            const long long e = (long long)r * p.cols + c;
            v = load4((const T*)p.x + e, n);
            if constexpr (STEP) {
                const f32x4 m = load4(p.momentum + e, n);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = k < n ? direction(v[k], m[k], mu, nesterov) : 0.f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = (float)((double)v[k] * factor);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) tile[y + 16 * i][x + k] = v[k];
        if (r < p.rows && c < wide_c) pack4<TWO, FP16>(straight + r * lds_, c, v);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = c0 + y + 16 * i, r = r0 + x;
        if (c < p.cols && r < wide_r) {
            f32x4 v;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = tile[x + k][y + 16 * i];
            pack4<TWO, FP16>(turned + c * ldt, r, v);
        }
    }
}

// tile `id` of the lower triangle, row by row
__device__ __forceinline__ void triangle_of(int id, int& tm, int& tn) {
    tm = (int)((sqrtf(8.f * (float)id + 1.f) - 1.f) * 0.5f);
    while (tm * (tm + 1) / 2 > id) --tm;
    while ((tm + 1) * (tm + 2) / 2 <= id) ++tm;
    tn = id - tm * (tm + 1) / 2;
}

// a tile of a symmetric matrix [m][packed m], value(i, j) being its numbers, and (off the diagonal) its mirror
template <class TileT, class F>
__device__ __forceinline__ void symmetric_store(TileT& T, char* lds, u16* __restrict__ p, long long ld, int m, int tm, int tn, F&& value) {
    const int wide = (int)(ld / 2);
#pragma unroll
    for (int i = 0; i < TileT::MI; ++i)
#pragma unroll
        for (int j = 0; j < TileT::NI; ++j) {
            const int row = tm * TileT::BM + TileT::row(i), col = tn * TileT::BN + TileT::col(j);
            if (row < m && col < wide) pack4<TWO, FP16>(p + row * ld, col, value(i, j));
        }
    if (tm != tn) T.store_transposed(lds, p, ld, m, ld, tm * TileT::BM, tn * TileT::BN, value);
}

// ---- S = X X^T: lower tiles.  A problem of one share writes S, one of several leaves fp32 tiles for join_kernel.  Bound by the matrix
// instructions: 4096 x 4096 175 to 183 us = 1130 to 1180 TFLOP/s of fp16 products (three for one of
// fp32)
template <class TileT>
__global__ __launch_bounds__(TileT::THREADS, 2) void square_kernel(const Problem* __restrict__ table, const int* __restrict__ ends, int count,
        const int* __restrict__ classes, Exponents ex, char* __restrict__ ws) {
    UNFLOW_DYNAMIC_LDS(char, lds);
    int id, tm, tn;
    const Problem p = table[dealt_problem_of(ends, count, classes, id)];
    triangle_of(id / p.shares, tm, tn);
    const int share = id % p.shares;
    const long long ld = packed_width(TWO, p.n), lds_ = packed_width(TWO, p.m);
    const int stages = ceil_div((int)ld, 64), per = ceil_div(stages, p.shares);
    const int k0 = share * per * 64, k1 = (share + 1) * per * 64 < (int)ld ? (share + 1) * per * 64 : (int)ld;
    const Operand X{(const u16*)(ws + p.X), ld, p.m};
    TileT T;
    T.run(X, X, k0, k1, tm * TileT::BM, tn * TileT::BN, lds);
    if (p.shares > 1) {
        float* to = (float*)(ws + p.shares_at) + (long long)id * (TileT::BM * TileT::BN);
#pragma unroll
        for (int i = 0; i < TileT::MI; ++i)
#pragma unroll
            for (int j = 0; j < TileT::NI; ++j) *reinterpret_cast<f32x4*>(to + TileT::row(i) * TileT::BN + TileT::col(j)) = T.acc[i][j];
        return;
    }
    const float f = ldexpf(1.f, ex.s - 2 * ex.x);
    symmetric_store(T, lds, (u16*)(ws + p.S), lds_, p.m, tm, tn, [&](int i, int j) { return T.acc[i][j] * f; });
}
// (64 x 64 of a tile of side `size` per workgroup; 5 to 7 us, the latency of a launch and of its loads)
__global__ __launch_bounds__(256) void join_kernel(const Problem* __restrict__ table, const int* __restrict__ ends, int count, int size,
        Exponents ex, char* __restrict__ ws) {
    __shared__ float tile[64][65];
    int id, tm, tn;
    const Problem p = table[problem_of(ends, count, (int)blockIdx.x, id)];
    const int side = size / 64, part = id % (side * side), at = id / (side * side);
    triangle_of(at, tm, tn);
    const int r0 = part / side * 64, c0 = part % side * 64, row0 = tm * size + r0, col0 = tn * size + c0;
    const long long each = (long long)size * size, ld = packed_width(TWO, p.m);
    const float* from = (const float*)(ws + p.shares_at) + at * p.shares * each + r0 * size + c0;
    u16* S = (u16*)(ws + p.S);
    const float f = ldexpf(1.f, ex.s - 2 * ex.x);
    const int x = (threadIdx.x & 15) * 4, y = threadIdx.x >> 4, wide = (int)(ld / 2);
    f32x4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const f32x4*>(from + (y + 16 * i) * size + x);
    for (int s = 1; s < p.shares; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += *reinterpret_cast<const f32x4*>(from + s * each + (y + 16 * i) * size + x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] *= f;
        const int row = row0 + y + 16 * i, col = col0 + x;
        if (row < p.m && col < wide) pack4<TWO, FP16>(S + row * ld, col, v[i]);
#pragma unroll
        for (int k = 0; k < 4; ++k) tile[y + 16 * i][x + k] = v[i][k];
    }
    __syncthreads();
    if (tm == tn) return;                                            // (a tile on the diagonal holds its own mirror)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = col0 + y + 16 * i, col = row0 + x;
        if (row < p.m && col < wide) {
            f32x4 u;
#pragma unroll
            for (int k = 0; k < 4; ++k) u[k] = tile[x + k][y + 16 * i];
            pack4<TWO, FP16>(S + row * ld, col, u);
        }
    }
}

// ---- Q = a I + b S + c S S: lower tiles.  Bound by the matrix instructions: 4096 x 4096 182 to 190 us
template <class TileT>
__global__ __launch_bounds__(TileT::THREADS, 2) void poly_kernel(const Problem* __restrict__ table, const int* __restrict__ ends, int count,
        const int* __restrict__ classes, float a, float b, float c, Exponents ex,
        char* __restrict__ ws) {
    UNFLOW_DYNAMIC_LDS(char, lds);
    int id, tm, tn;
    const Problem p = table[dealt_problem_of(ends, count, classes, id)];
    triangle_of(id, tm, tn);
    const long long ld = packed_width(TWO, p.m);
    const u16* s = (const u16*)(ws + p.S);
    const Operand S{s, ld, p.m};
    TileT T;
    T.run(S, S, 0, (int)ld, tm * TileT::BM, tn * TileT::BN, lds);
    const float fb = ldexpf(b, ex.q - ex.s), fc = ldexpf(c, ex.q - 2 * ex.s), fa = ldexpf(a, ex.q);
    const int wide = (int)(ld / 2);
#pragma unroll
    for (int i = 0; i < TileT::MI; ++i)
#pragma unroll
        for (int j = 0; j < TileT::NI; ++j) {
            const int row = tm * TileT::BM + TileT::row(i), col = tn * TileT::BN + TileT::col(j);
            if (row >= p.m || col >= wide) continue;                   // (what is not there is zero already)
            const f32x4 v = unpack4<TWO, FP16>(s + row * ld, col);
#pragma unroll
            for (int r = 0; r < 4; ++r) T.acc[i][j][r] = fmaf(fc, T.acc[i][j][r], fb * v[r]) + (row == col + r ? fa : 0.f);
        }
    symmetric_store(T, lds, (u16*)(ws + p.Q), ld, p.m, tm, tn, [&](int i, int j) { return T.acc[i][j]; });
}

// ---- X <- Q X.  LAST: the output, or the parameter's update.  Bound by the matrix instructions (4096 x 4096 306 to 317 us = 1300 to 1350 TFLOP/s
// of fp16 products), for the weights above as much by writing X both ways (315 us = 980 TFLOP/s, 400 MB written): S sums over the columns of X and the next
// X over its rows, and both operands of a product lie along what is summed
struct Update { float keep, lr; };                                   // 1 - lr wd, lr
template <class TileT, bool LAST, bool STEP, class T>
__global__ __launch_bounds__(TileT::THREADS, 2) void apply_kernel(const Problem* __restrict__ table, const int* __restrict__ ends, int count,
        const int* __restrict__ classes, int odd, Exponents ex, Update up,
        char* __restrict__ ws) {
    UNFLOW_DYNAMIC_LDS(char, lds);
    int id, tm, tn;
    const Problem p = table[dealt_problem_of(ends, count, classes, id)];
    tile_of(id, ceil_div(p.m, TileT::BM), ceil_div(p.n, TileT::BN), tm, tn);
    const long long ldm = packed_width(TWO, p.m), ldn = packed_width(TWO, p.n);
    const Operand Q{(const u16*)(ws + p.Q), ldm, p.m}, XT{(const u16*)(ws + (odd ? p.XT1 : p.XT0)), ldm, p.n};
    TileT T_;
    T_.run(Q, XT, 0, (int)ldm, tm * TileT::BM, tn * TileT::BN, lds);
    const float f = ldexpf(1.f, LAST ? -(ex.q + ex.x) : -ex.q);
    const int wide_n = (int)(ldn / 2);
    u16 *X = (u16*)(ws + p.X), *next = (u16*)(ws + (odd ? p.XT0 : p.XT1));
    const bool tall = p.rows > p.cols;
    const float lr = up.lr * p.boost;
#pragma unroll
    for (int i = 0; i < TileT::MI; ++i)
#pragma unroll
        for (int j = 0; j < TileT::NI; ++j) {
            const int row = tm * TileT::BM + TileT::row(i), col = tn * TileT::BN + TileT::col(j);
            f32x4 v = T_.acc[i][j] *= f;
            if constexpr (LAST) {
                if (row >= p.m || col >= p.n) continue;
                const int n = p.n - col < 4 ? p.n - col : 4;
                T* out = (T*)p.out;
                if (!tall) {
                    out += (long long)row * p.cols + col;
                    if constexpr (STEP) v = load4(out, n) * up.keep - v * lr;
                    store4<T>(out, v, n);
                } else {
                    out += (long long)col * p.cols + row;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (r < n) {
                            T* o = out + (long long)r * p.cols;
                            *o = (T)(STEP ? (float)*o * up.keep - v[r] * lr : v[r]);
                        }
                }
            } else if (row < p.m && col < wide_n) pack4<TWO, FP16>(X + row * ldn, col, v);
        }
    __builtin_amdgcn_sched_barrier(0);                                // (the addresses of both stores at once do not fit the registers)
    if constexpr (!LAST) T_.store_transposed(lds, next, ldm, p.n, ldm, tm * TileT::BM, tn * TileT::BN, [&](int i, int j) { return T_.acc[i][j]; });
}

// ---- matrices of up to 32 rows (or columns).  All X of the iteration are polynomials in S_0 = X_0 X_0^T times X_0, so it can run on m x m matrices:
//   P <- Q P,  S <- Q S Q,  Q = a I + b S + c S S;   X = P X_0 at the end
// one read of the matrix for S_0, whose trace is the squared norm, and one for the result: 3 launches instead of 22.  Squaring the singular values
// needs twice the digits (what rounding adds to S_0 is multiplied by a^10), so all sums are 64 bits, and that is what bounds m: the 17 products
// of one workgroup take 17 m^3 fused operations at 64 a cycle (18 us for m = 32).  8 x 500: 30 us against 50 by the tiles, 8 of 32 x 1152 44 against
// 98, 32 x 100000 122 against 382; and nearer to the formula than the tiles' planes, whose two roundings a step show where sums are short (4 x 512:
// 3.5e-6 by the tiles, 1.5e-6 in fp32).  Rounding leaves S_0 directions of slightly negative size where the matrix has none; they grow by |a^2| a step,
// and nothing holds them once they are no longer small (below zero the polynomial has no bound), so a list goes here only for as many steps as keep
// them below 2^-10 (narrow_holds; 9 with the default coefficients).  Beyond, and in the tiles' own iteration, S is a product X X^T at every
// step and cannot leave zero by more than its rounding.  A list that has larger matrices goes by the tiles as a whole, whose launches are there anyhow (the flow
// network's weights: 252 us, 299 where those of few rows have their own kernels).
constexpr int kNarrow = 32, kColumns = 128, kGramParts = 64;         // a workgroup takes 128 columns at a time; S_0 is summed in at most 64 parts
constexpr int kNarrowNumbers = kNarrow * kColumns / 256;             // of a thread

// the columns j0 .. of a matrix as they lie in memory: number q of a thread is (i, j), j < width where there is one
struct Columns {
    int m, n, j0, width;
    bool tall;
    __device__ __forceinline__ Columns(const Problem& p, int chunk)
        : m(p.m), n(p.n), j0(chunk * kColumns), width(p.n - chunk * kColumns < kColumns ? p.n - chunk * kColumns : kColumns), tall(p.rows > p.cols) {}
    __device__ __forceinline__ void place(int q, int& i, int& j) const {
        const int e = q * 256 + (int)threadIdx.x;
        const bool in_rows = tall && e < kColumns * m;               // (behind the last number both give rows m ..)
        i = in_rows ? e % m : e / kColumns;
        j = in_rows ? e / m : e % kColumns;
    }
    __device__ __forceinline__ bool there(int i, int j) const { return i < m && j < width; }
    __device__ __forceinline__ long long at(int i, int j) const { return tall ? (long long)(j0 + j) * m + i : (long long)i * n + j0 + j; }
};
typedef float NarrowTile[kColumns + 4] __attribute__((aligned(16)));

// the update's direction (or the matrix) into x [32][128]; zeros where nothing is.  FIRST: the momentum is brought up to date
template <class T, bool STEP, bool FIRST>
__device__ __forceinline__ void load_columns(const Problem& p, const Columns& c, float mu, int nesterov, NarrowTile* x) {
    float v[kNarrowNumbers], m[kNarrowNumbers];
#pragma unroll
    for (int q = 0; q < kNarrowNumbers; ++q) {
        int i, j;
        c.place(q, i, j);
        v[q] = c.there(i, j) ? load1((const T*)p.x + c.at(i, j)) : 0.f;
        m[q] = STEP && c.there(i, j) ? p.momentum[c.at(i, j)] : 0.f;
    }
#pragma unroll
    for (int q = 0; q < kNarrowNumbers; ++q) {
        int i, j;
        c.place(q, i, j);
        if constexpr (STEP) {
            if constexpr (FIRST) {
                m[q] = m[q] + (1.f - mu) * (v[q] - m[q]);
                if (c.there(i, j)) p.momentum[c.at(i, j)] = m[q];
            }
            v[q] = direction(v[q], m[q], mu, nesterov);
        }
        x[i][j] = v[q];
    }
}

// a part of S_0 |G|^2: a thread sums 2 x 2 numbers in 64 bits (products of 32-bit numbers are exact)
template <class T, bool STEP>
__global__ __launch_bounds__(256) void narrow_gram_kernel(const Problem* __restrict__ table, const int* __restrict__ ends, int count, float mu,
        int nesterov, char* __restrict__ ws) {
    __shared__ NarrowTile x[kNarrow];
    int part;
    const Problem p = table[problem_of(ends, count, (int)blockIdx.x, part)];
    const int chunks = ceil_div(p.n, kColumns), per = ceil_div(chunks, p.parts), last = (part + 1) * per < chunks ? (part + 1) * per : chunks;
    const int i = 2 * ((int)threadIdx.x >> 4), k = 2 * ((int)threadIdx.x & 15);
    double s[2][2] = {};
    for (int c = part * per; c < last; ++c) {
        load_columns<T, STEP, true>(p, Columns(p, c), mu, nesterov, x);
        __syncthreads();
        if (i < p.m && k < p.m)
#pragma unroll 4
            for (int j = 0; j < kColumns; j += 4) {
                const f32x4 a[2] = {*reinterpret_cast<const f32x4*>(&x[i][j]), *reinterpret_cast<const f32x4*>(&x[i + 1][j])};
                const f32x4 b[2] = {*reinterpret_cast<const f32x4*>(&x[k][j]), *reinterpret_cast<const f32x4*>(&x[k + 1][j])};
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int w = 0; w < 2; ++w) s[u][w] = fma((double)a[u][q], (double)b[w][q], s[u][w]);
            }
        __syncthreads();
    }
    double* to = (double*)(ws + p.S) + (long long)part * kNarrow * kNarrow;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int w = 0; w < 2; ++w) to[(i + u) * kNarrow + k + w] = s[u][w];
}

typedef double f64x2 __attribute__((ext_vector_type(2)));
typedef double NarrowMatrix[kNarrow + 2] __attribute__((aligned(16)));
// a thread's 2 x 2 numbers of A B for symmetric matrices (B's columns are its rows), zeros behind m
__device__ __forceinline__ void narrow_product(const NarrowMatrix* A, const NarrowMatrix* B, int m, int i, int k, double (&c)[2][2]) {
    double s[2][2] = {};
    for (int q = 0; q < m; q += 2) {
        const f64x2 a[2] = {*reinterpret_cast<const f64x2*>(&A[i][q]), *reinterpret_cast<const f64x2*>(&A[i + 1][q])};
        const f64x2 b[2] = {*reinterpret_cast<const f64x2*>(&B[k][q]), *reinterpret_cast<const f64x2*>(&B[k + 1][q])};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int w = 0; w < 2; ++w) s[u][w] = fma(a[u].y, b[w].y, fma(a[u].x, b[w].x, s[u][w]));
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int w = 0; w < 2; ++w) c[u][w] = s[u][w];
}

// S_0 from its parts, in order, and P / (norm + eps), 1024 numbers at p.Q.  A workgroup per matrix
__global__ __launch_bounds__(256) void narrow_iterate_kernel(const Problem* __restrict__ table, int steps, double a, double b, double c, float eps,
        char* __restrict__ ws) {
    __shared__ NarrowMatrix S[kNarrow], Q[kNarrow], P[kNarrow];
    const Problem p = table[blockIdx.x];
    const int i = 2 * ((int)threadIdx.x >> 4), k = 2 * ((int)threadIdx.x & 15), m = p.m;
    const bool in = i < m && k < m;
    double v[2][2] = {}, mine[2][2];
    auto put = [&](NarrowMatrix* to, double scale) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int w = 0; w < 2; ++w) to[i + u][k + w] = v[u][w] * scale;
    };
    const double* parts = (const double*)(ws + p.S) + i * kNarrow + k;
#pragma unroll 4
    for (int q = 0; q < p.parts; ++q) {
        const f64x2 x = *reinterpret_cast<const f64x2*>(parts + (long long)q * kNarrow * kNarrow);
        const f64x2 y = *reinterpret_cast<const f64x2*>(parts + (long long)q * kNarrow * kNarrow + kNarrow);
        v[0][0] += x.x; v[0][1] += x.y; v[1][0] += y.x; v[1][1] += y.y;
    }
    put(S, 1.);
    __syncthreads();
    double trace = 0.;
    for (int q = 0; q < m; ++q) trace += S[q][q];
    const double factor = 1. / (sqrt(trace) + (double)eps);
    __syncthreads();
    put(S, factor * factor);
    __syncthreads();
    for (int step = 0; step < steps; ++step) {
        if (in) {
            narrow_product(S, S, m, i, k, v);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int w = 0; w < 2; ++w) v[u][w] = c * v[u][w] + b * S[i + u][k + w] + (i + u == k + w && i + u < m ? a : 0.);
        }
        put(Q, 1.);
        __syncthreads();
        if (step == 0) put(P, 1.);
        else {
            if (in) narrow_product(Q, P, m, i, k, v);
            __syncthreads();
            put(P, 1.);
        }
        if (step + 1 < steps) {
            if (in) narrow_product(Q, S, m, i, k, v);
            __syncthreads();
            put(S, 1.);
            __syncthreads();
            if (in) narrow_product(Q, S, m, i, k, mine);
            __syncthreads();
            if (in)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int w = 0; w < 2; ++w) S[i + u][k + w] = mine[u][w];
        }
        __syncthreads();
    }
    double* to = (double*)(ws + p.Q);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int w = 0; w < 2; ++w) to[(i + u) * kNarrow + k + w] = P[i + u][k + w] * factor;
}

// X = P X_0 of 128 columns: a thread has one column and half of the rows.  The output, or the parameter's update
template <class T, bool STEP>
__global__ __launch_bounds__(256) void narrow_apply_kernel(const Problem* __restrict__ table, const int* __restrict__ ends, int count, float mu,
        int nesterov, Update up, const char* __restrict__ ws) {
    __shared__ NarrowTile x[kNarrow];
    __shared__ NarrowMatrix P[kNarrow];
    int chunk;
    const Problem p = table[problem_of(ends, count, (int)blockIdx.x, chunk)];
    const double* from = (const double*)(ws + p.Q);
    for (int e = (int)threadIdx.x; e < kNarrow * kNarrow; e += 256) P[e / kNarrow][e % kNarrow] = from[e];
    const Columns c(p, chunk);
    load_columns<T, STEP, false>(p, c, mu, nesterov, x);
    __syncthreads();
    const int j = (int)threadIdx.x & (kColumns - 1), r0 = (int)threadIdx.x / kColumns * 16;
    f64x2 v[8] = {};
    if (r0 < p.m)
        for (int k = 0; k < p.m; ++k) {
            const double xk = (double)x[k][j];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const f64x2 pk = *reinterpret_cast<const f64x2*>(&P[k][r0 + 2 * r]);
                v[r] = f64x2{fma(pk.x, xk, v[r].x), fma(pk.y, xk, v[r].y)};
            }
        }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r0 + r][j] = (float)v[r / 2][r % 2];
    __syncthreads();
    const float lr = up.lr * p.boost;
    T* out = (T*)p.out;
    float old[kNarrowNumbers];
#pragma unroll
    for (int q = 0; q < kNarrowNumbers; ++q) {
        int i, k;
        c.place(q, i, k);
        old[q] = STEP && c.there(i, k) ? load1(out + c.at(i, k)) : 0.f;
    }
#pragma unroll
    for (int q = 0; q < kNarrowNumbers; ++q) {
        int i, k;
        c.place(q, i, k);
        if (c.there(i, k)) out[c.at(i, k)] = (T)(STEP ? old[q] * up.keep - x[i][k] * lr : x[i][k]);
    }
}

// ---- the host side
template <class F> static void with_tile(int size, F&& f) {
    if (size == 0) f(Tile<256, 256, 2, 4, 2, TWO, FP16>{});
    else if (size == 1) f(Tile<192, 192, 2, 4, 3, TWO, FP16>{});
    else if (size == 2) f(Tile<128, 128, 2, 2, 2, TWO, FP16>{});
    else if (size == 3) f(Tile<64, 64, 2, 2, 2, TWO, FP16>{});
    else if (size == 4) f(Tile<128, 128, 2, 2, 4, TWO, FP16>{});
    else f(Tile<64, 64, 2, 2, 4, TWO, FP16>{});
}

// Bounds of |X|, |S|, |Q| (spectral norms: every singular value of X_0 is in [0, 1]) over all steps, as powers of two that keep the planes
// below 2^15 with a quarter to spare.  false: the iteration leaves [0, 16] and is of no use.
static bool exponents_of(int steps, float a, float b, float c, Exponents& ex) {
    double mx = 1., ms = 1., mq = 1.;
    for (int i = 0; i <= 512; ++i) {
        double s = i / 512.;
        for (int k = 0; k < steps; ++k) {
            const double t = s * s, q = fabs(a + b * t + c * t * t);
            mq = mq > q ? mq : q;
            s *= q;
            if (!(s <= 16.)) return false;
            mx = mx > s ? mx : s;
        }
    }
    ms = mx * mx;
    if (!(mq <= 4096.)) return false;
    auto exponent = [](double v) { int e = 15; while (v * 1.25 > 1.) { v *= 0.5; --e; } return e; };
    ex = Exponents{exponent(mx), exponent(ms), exponent(mq)};
    return true;
}

// log2 of how much `steps` times S <- Q S Q make of a small error in S at most: the largest |d (s q(s)^2) / ds| over the squares of all singular
// values, to the power of `steps` (at s = 0, a direction the matrix does not have, it is a^2).  -1: the singular values leave [0, 16].
static double growth_of(int steps, double a, double b, double c) {
    double most = 0., top = 1.;
    for (int k = 0; k <= steps; ++k) {                                   // the singular values after k steps lie in [0, top]
        double next = 0.;
        for (int i = 0; i <= 64; ++i) {
            const double s = top * i / 64., t = s * s, q = a + b * t + c * t * t, slope = fabs(q * q + 2. * t * q * (b + 2. * c * t));
            most = most > slope ? most : slope;
            next = next > s * fabs(q) ? next : s * fabs(q);
        }
        if (next <= top && k > 0) break;                                 // (nothing new from here on)
        top = top > next ? top : next;
        if (!(top <= 16.)) return -1.;
    }
    return most > 1. ? steps * log2(most) : 0.;
}

constexpr long long kGroupBytes = 4ll << 30;                         // matrices are taken together as long as their planes fit in this

struct Group {
    int first, count;                                                // of the list
    bool narrow;                                                     // all of few rows
    int grams, columns;                                              // the work items of the kernels for these
    int size_s, size_q, size_x;                                      // indices into kSizes
    // numbers a workgroup of the norm takes: few of a small list, so that it fills the chip
    int chunk;
    int total[kPhases];
    long long table, ends, parts, table_bytes, bytes;
};

static long long plane_bytes(long long m, long long n) {
    const long long wm = packed_width(TWO, m), wn = packed_width(TWO, n);
    return round_up(2 * wn * m, 256) + 2 * round_up(2 * wm * n, 256) + 2 * round_up(2 * wm * m, 256);
}

constexpr int kMost = 1024;                                          // matrices of one group

// the matrices [first, first + count) of a list, sorted by the longer side and then the shorter one, the largest first
struct Sorted {
    int at[kMost];
    int m[kMost], n[kMost];
};
static void sort_of(const unflow_matrix* a, int first, int count, Sorted& s) {
    for (int i = 0; i < count; ++i) s.at[i] = first + i;
    auto side = [&](int i, bool longer) { return (a[i].rows < a[i].cols) == longer ? a[i].cols : a[i].rows; };
    std::stable_sort(s.at, s.at + count, [&](int x, int y) {
        const int nx = side(x, true), ny = side(y, true);
        return nx != ny ? nx > ny : side(x, false) > side(y, false);
    });
    for (int i = 0; i < count; ++i) {
        s.m[i] = side(s.at[i], false);
        s.n[i] = side(s.at[i], true);
    }
}

static Problem problem_for(const unflow_matrix& q, int m, int n) {
    Problem p{};
    p.x = q.x; p.out = q.out; p.momentum = q.momentum;
    p.rows = q.rows; p.cols = q.cols;
    p.m = m; p.n = n;
    p.boost = q.rows > q.cols ? sqrtf((float)q.rows / (float)q.cols) : 1.f;
    return p;
}

// Whether matrices of up to m <= n numbers a side may take the kernels for few rows, where an error in S grows by 2^growth.  S_0 is off by a rounding
// for each number that is summed after another (the columns of a part and its chunks, then the parts), a step adds the roundings of three products
// of m terms; all of it has to stay below 2^-10 of a singular value of 1.
static bool narrow_holds(int m, int n, double growth) {
    const int chunks = ceil_div(n, kColumns), parts = chunks < kGramParts ? chunks : kGramParts;
    return m <= kNarrow && log2((double)ceil_div(chunks, parts) * kColumns + parts + 4. * m) - 53. + growth <= -10.;
}

// lays out a group: problems and running counts on the host (`table`: what g.table_bytes of the workspace will hold), offsets into the workspace
static Group lay_out(const unflow_matrix* a, int first, int count, double growth, char* table) {
    static thread_local Sorted order;
    static thread_local Job jobs[kMost];
    sort_of(a, first, count, order);
    Group g{};
    g.first = first;
    g.count = count;
    g.narrow = narrow_holds(*std::max_element(order.m, order.m + count), order.n[0], growth);
    long long at = 0, chunks = 0;
    auto take = [&](long long bytes) { const long long p = at; at += round_up(bytes, 256); return p; };
    g.ends = (long long)sizeof(Problem) * count;                     // (of the table)
    g.table_bytes = g.ends + 4ll * (g.narrow ? 2 : kTables) * count;
    g.table = take(g.table_bytes);
    Problem* problems = (Problem*)table;
    int* ends = (int*)(table ? table + g.ends : nullptr);
    if (g.narrow) {
        for (int i = 0; i < count; ++i) {
            Problem p = problem_for(a[order.at[i]], order.m[i], order.n[i]);
            const int columns = ceil_div(p.n, kColumns);
            p.parts = columns < kGramParts ? columns : kGramParts;
            p.S = take(8ll * kNarrow * kNarrow * p.parts);
            p.Q = take(8ll * kNarrow * kNarrow);
            g.grams += p.parts;
            g.columns += columns;
            if (table) {
                problems[i] = p;
                ends[i] = g.grams;
                ends[count + i] = g.columns;
            }
        }
        g.bytes = at;
        return g;
    }
    // matrices of one shape are one job of the model
    auto plan = [&](auto job_of) {
        int k = 0;
        for (int i = 0; i < count;) {
            int e = i + 1;
            while (e < count && order.m[e] == order.m[i] && order.n[e] == order.n[i]) ++e;
            jobs[k] = job_of(order.m[i], order.n[i]);
            jobs[k++].times = e - i;
            i = e;
        }
        return choose(TWO, jobs, k);
    };
    const Choice cs = plan([](long long m, long long n) { return Job{m, m, stages_of(packed_width(TWO, n)), true, true, 8.}; });
    g.size_s = cs.size;
    g.size_q = plan([](long long m, long long n) { return Job{m, m, stages_of(packed_width(TWO, m)), true, false, 8.}; }).size;
    g.size_x = plan([](long long m, long long n) { return Job{m, n, stages_of(packed_width(TWO, m)), false, false, 8.}; }).size;
    long long numbers = 0;
    for (int i = 0; i < count; ++i) numbers += (long long)order.m[i] * order.n[i];
    g.chunk = numbers < (16 << 20) ? 4096 : 16384;
    for (int i = 0; i < count; ++i) chunks += ((long long)order.m[i] * order.n[i] + g.chunk - 1) / g.chunk;
    g.parts = take(8 * chunks);
    int part0 = 0, run[kPhases] = {};
    for (int i = 0; i < count; ++i) {
        Problem p = problem_for(a[order.at[i]], order.m[i], order.n[i]);
        p.X = take(2 * packed_width(TWO, p.n) * p.m);
        p.XT0 = take(2 * packed_width(TWO, p.m) * p.n);
        p.XT1 = take(2 * packed_width(TWO, p.m) * p.n);
        p.S = take(2 * packed_width(TWO, p.m) * p.m);
        p.Q = take(2 * packed_width(TWO, p.m) * p.m);
        p.shares = shares_of(stages_of(packed_width(TWO, p.n)), cs.limit);
        const int low = (int)lower_tiles_of(p.m, kSizes[g.size_s]);
        if (p.shares > 1) p.shares_at = take(4ll * kSizes[g.size_s] * kSizes[g.size_s] * low * p.shares);
        p.part0 = part0;
        p.parts = (int)(((long long)p.rows * p.cols + g.chunk - 1) / g.chunk);
        part0 += p.parts;
        run[kNorm] += p.parts;
        run[kPack] += ceil_div(p.rows, 64) * ceil_div(p.cols, 64);
        run[kSquare] += low * p.shares;
        run[kJoin] += p.shares > 1 ? low * (kSizes[g.size_s] / 64) * (kSizes[g.size_s] / 64) : 0;
        run[kPoly] += (int)lower_tiles_of(p.m, kSizes[g.size_q]);
        run[kApply] += (int)tiles_of(p.m, p.n, kSizes[g.size_x]);
        if (table) {
            problems[i] = p;
            for (int k = 0; k < kPhases; ++k) ends[k * count + i] = run[k];
        }
    }
    if (table) {
        // matrices whose work items of a phase are equally long are dealt out together (they are neighbours for S, which sums over n; the other two
        // sum over m, which need not be in order: as far as neighbours are alike)
        const int phases[3] = {kSquare, kPoly, kApply}, tables[3] = {kSquareClass, kPolyClass, kApplyClass};
        for (int k = 0; k < 3; ++k)
            for (int i = 0; i < count;) {
                int e = i + 1;
                while (e < count && (k == 0 ? order.n[e] == order.n[i] && problems[e].shares == problems[i].shares : order.m[e] == order.m[i])) ++e;
                const int* run_of = ends + phases[k] * count;
                for (int j = i; j < e; ++j) {
                    ends[tables[k] * count + 2 * j] = i ? run_of[i - 1] : 0;
                    ends[tables[k] * count + 2 * j + 1] = run_of[e - 1];
                }
                i = e;
            }
    }
    for (int k = 0; k < kPhases; ++k) g.total[k] = run[k];
    g.bytes = at;
    return g;
}
static int group_end(const unflow_matrix* a, int count, int first) {
    long long bytes = 0;
    int i = first;
    for (; i < count && i - first < kMost; ++i) {
        const long long r = a[i].rows, c = a[i].cols;
        bytes += plane_bytes(r < c ? r : c, r < c ? c : r);
        if (i > first && bytes > kGroupBytes) break;
    }
    return i;
}

static bool matrices_ok(const unflow_matrix* a, int count, int dtype) {
    if (!a || count <= 0 || dtype < kFp32 || dtype > kFp16) return false;
    for (int i = 0; i < count; ++i)
        if (a[i].rows <= 0 || a[i].cols <= 0 || a[i].rows > UNFLOW_MATRIX_MAX_SIDE || a[i].cols > UNFLOW_MATRIX_MAX_SIDE) return false;
    return true;
}

// Whether no parameter or momentum shares memory with another one, or with another weight's gradient: the kernels work on all of them at once.  (A
// weight's own gradient may be its momentum or its parameter: whoever writes a number has read it.)  false, too, without memory for the list.
static bool apart(const unflow_matrix* a, int count, int dtype) {
    struct Span { size_t from, to; bool written; };
    const size_t size = dtype == kFp32 ? 4 : 2;
    Span* spans = (Span*)malloc(sizeof(Span) * 3 * (size_t)count);
    if (!spans) return false;
    int n = 0;
    for (int i = 0; i < count; ++i) {
        const size_t numbers = (size_t)a[i].rows * (size_t)a[i].cols, g = (size_t)a[i].x, p = (size_t)a[i].out, m = (size_t)a[i].momentum;
        spans[n++] = Span{p, p + numbers * size, true};
        spans[n++] = Span{m, m + numbers * 4, true};
        if (g != p && (g != m || size != 4)) spans[n++] = Span{g, g + numbers * size, false};
    }
    std::sort(spans, spans + n, [](const Span& x, const Span& y) { return x.from < y.from; });
    size_t written = 0, read = 0;                                        // bytes behind what lies before
    bool good = true;
    for (int i = 0; i < n && good; ++i) {
        good = spans[i].from >= written && !(spans[i].written && spans[i].from < read);
        size_t& reach = spans[i].written ? written : read;
        reach = reach > spans[i].to ? reach : spans[i].to;
    }
    free(spans);
    return good;
}

#define LAUNCH_TILES(kernel, count, ...)                                                                                              \
    do {                                                                                                                              \
        if (TileT::LDS > 65536) (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, TileT::LDS); \
        UNFLOW_LAUNCH(kernel, dim3(count), dim3(TileT::THREADS), TileT::LDS, stream, __VA_ARGS__);                                    \
    } while (0)

static void write_table(const void* src, long long bytes, char* dst, hipStream_t stream) {
    for (long long at = 0; at < bytes; at += sizeof(Words)) {
        Words w;
        const long long n = bytes - at < (long long)sizeof(Words) ? bytes - at : (long long)sizeof(Words);
        memcpy(w.w, (const char*)src + at, n);
        UNFLOW_LAUNCH(write_table_kernel, dim3(1), dim3(256), 0, stream, w, (int)(n / 4), (unsigned*)(dst + at));
    }
}

template <class T, bool STEP>
static void iterate(const Group& g, int steps, float a, float b, float c, float eps, float mu, int nesterov, Update up, Exponents ex, char* ws,
        hipStream_t stream) {
    const Problem* table = (const Problem*)(ws + g.table);
    const int* ends = (const int*)(ws + g.table + g.ends);
    const int n = g.count;
    if (g.narrow) {
        UNFLOW_LAUNCH((narrow_gram_kernel<T, STEP>), dim3(g.grams), dim3(256), 0, stream, table, ends, n, mu, nesterov, ws);
        UNFLOW_LAUNCH(narrow_iterate_kernel, dim3(n), dim3(256), 0, stream, table, steps, (double)a, (double)b, (double)c, eps, ws);
        UNFLOW_LAUNCH((narrow_apply_kernel<T, STEP>), dim3(g.columns), dim3(256), 0, stream, table, ends + n, n, mu, nesterov, up, (const char*)ws);
        return;
    }
    double* parts = (double*)(ws + g.parts);
    UNFLOW_LAUNCH((norm_kernel<T, STEP>), dim3(g.total[kNorm]), dim3(256), 0, stream, table, ends + kNorm * n, n, g.chunk, mu, nesterov, parts);
    UNFLOW_LAUNCH((start_kernel<T, STEP>), dim3(g.total[kPack]), dim3(256), 0, stream, table, ends + kPack * n, n, (const double*)parts, mu,
        nesterov, eps, ex, ws);
    for (int k = 0; k < steps; ++k) {
        with_tile(g.size_s, [&](auto tile) {
            using TileT = decltype(tile);
            LAUNCH_TILES((square_kernel<TileT>), g.total[kSquare], table, ends + kSquare * n, n, ends + kSquareClass * n, ex, ws);
        });
        if (g.total[kJoin]) UNFLOW_LAUNCH(join_kernel, dim3(g.total[kJoin]), dim3(256), 0, stream, table, ends + kJoin * n, n, kSizes[g.size_s], ex,
            ws);
        with_tile(g.size_q, [&](auto tile) {
            using TileT = decltype(tile);
            LAUNCH_TILES((poly_kernel<TileT>), g.total[kPoly], table, ends + kPoly * n, n, ends + kPolyClass * n, a, b, c, ex, ws);
        });
        with_tile(g.size_x, [&](auto tile) {
            using TileT = decltype(tile);
            if (k + 1 < steps) LAUNCH_TILES((apply_kernel<TileT, false, false, float>), g.total[kApply], table, ends + kApply * n, n,
                ends + kApplyClass * n, k & 1, ex, up, ws);
            else LAUNCH_TILES((apply_kernel<TileT, true, STEP, T>), g.total[kApply], table, ends + kApply * n, n, ends + kApplyClass * n, k & 1, ex,
                up, ws);
        });
    }
}

static long long workspace_of(const unflow_matrix* a, int count, double growth) {
    long long most = 0;
    for (int i = 0; i < count;) {
        const int e = group_end(a, count, i);
        const long long b = lay_out(a, i, e - i, growth, nullptr).bytes;
        most = most > b ? most : b;
        i = e;
    }
    return most;
}

template <bool STEP>
static int run(const unflow_matrix* a, int count, int dtype, int steps, float ca, float cb, float cc, float eps, float mu, int nesterov, Update up,
        void* workspace, long long workspace_bytes, void* stream_) {
    Exponents ex;
    UNFLOW_REQUIRE(exponents_of(steps, ca, cb, cc, ex));
    const double growth = growth_of(steps, ca, cb, cc);
    UNFLOW_REQUIRE(growth >= 0. && workspace_bytes >= workspace_of(a, count, growth));
    hipStream_t stream = (hipStream_t)stream_;
    char* ws = (char*)workspace;
    for (int i = 0; i < count;) {
        const int e = group_end(a, count, i), n = e - i;
        static thread_local struct alignas(8) { char bytes[kMost * (sizeof(Problem) + 4 * kTables)]; } table;
        const Group g = lay_out(a, i, n, growth, table.bytes);
        write_table(table.bytes, g.table_bytes, ws + g.table, stream);
        if (dtype == kFp32) iterate<float, STEP>(g, steps, ca, cb, cc, eps, mu, nesterov, up, ex, ws, stream);
        else if (dtype == kBf16) iterate<__bf16, STEP>(g, steps, ca, cb, cc, eps, mu, nesterov, up, ex, ws, stream);
        else iterate<_Float16, STEP>(g, steps, ca, cb, cc, eps, mu, nesterov, up, ex, ws, stream);
        i = e;
    }
    return unflow_launch_status();
}

}  // namespace

extern "C" int unflow_orthogonalize_workspace(const unflow_matrix* matrices, int count, int dtype, long long* bytes) {
    UNFLOW_REQUIRE(bytes && matrices_ok(matrices, count, dtype));
    // (without and with so many steps that nothing goes by the kernels for few rows)
    *bytes = std::max(workspace_of(matrices, count, 0.), workspace_of(matrices, count, 1e3));
    return 0;
}

extern "C" int unflow_orthogonalize_workspace_ex(const unflow_matrix* matrices, int count, int dtype, int steps, float a, float b, float c,
        long long* bytes) {
    UNFLOW_REQUIRE(bytes && matrices_ok(matrices, count, dtype) && steps >= 1 && steps <= 64);
    const double growth = growth_of(steps, a, b, c);
    UNFLOW_REQUIRE(growth >= 0.);
    *bytes = workspace_of(matrices, count, growth);
    return 0;
}

extern "C" int unflow_orthogonalize(const unflow_matrix* matrices, int count, int dtype, int steps, float a, float b, float c, float eps,
        void* workspace, long long workspace_bytes, void* stream) {
    UNFLOW_REQUIRE(matrices_ok(matrices, count, dtype) && workspace && steps >= 1 && steps <= 64 && eps >= 0.f);
    for (int i = 0; i < count; ++i) UNFLOW_REQUIRE(matrices[i].x && matrices[i].out);
    return run<false>(matrices, count, dtype, steps, a, b, c, eps, 0.f, 0, Update{1.f, 0.f}, workspace, workspace_bytes, stream);
}

extern "C" int unflow_muon_step(const unflow_matrix* matrices, int count, int dtype, float lr, float momentum, float weight_decay, int nesterov,
        int steps, float a, float b, float c, float eps,
        void* workspace, long long workspace_bytes, void* stream) {
    UNFLOW_REQUIRE(matrices_ok(matrices, count, dtype) && workspace && steps >= 1 && steps <= 64 && eps >= 0.f);
    for (int i = 0; i < count; ++i) UNFLOW_REQUIRE(matrices[i].x && matrices[i].out && matrices[i].momentum);
    UNFLOW_REQUIRE(apart(matrices, count, dtype));
    return run<true>(matrices, count, dtype, steps, a, b, c, eps, momentum, nesterov, Update{1.f - lr * weight_decay, lr}, workspace,
        workspace_bytes, stream);
}
