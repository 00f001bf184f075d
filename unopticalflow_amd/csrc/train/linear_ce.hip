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
// fp32 inputs as two fp16 planes scaled by the largest magnitude (mfma16.h).  G keeps the type of the products: for bf16 inputs its rounding
// (2^-9 of every element, at random) is of the size of the gradients' own rounding; the uniform factors of G (scale, the upstream gradient of a
// reduced loss) are applied to the sums, so that -1 at the target stays exact.
//
// A row whose target is `ignore_index` has loss 0 and no gradient, whatever its hidden row holds (it is left out of the largest magnitude, and
// enters the transposed H as zeros: 0 * NaN never meets a sum).  Any other target outside [0, V) makes its row's loss and gradients NaN.
#include "pack.h"
#include <cmath>
#include <cstring>

namespace {

constexpr int kFp32 = 0, kBf16 = 1, kFp16 = 2;                     // UNFLOW_DTYPE_*
constexpr int kMaxima = 256;                                       // workgroups that look for the largest magnitude of one input

// Device scalars of one call.
struct Scalars {
    int eh, ew;                  // H and W are multiplied by 2^eh, 2^ew when they are packed
    float gmax;                  // largest finite |upstream| of the rows (reduction none), else 1
    float factor;                // the uniform factor of both gradients: scale, times the upstream gradient (sum), divided by the count (mean)
};

// ---- largest finite magnitude of W and of the rows of H that count (fp32 only): kMaxima workgroups each, one maximum per workgroup
__global__ __launch_bounds__(256) void largest_kernel(Source h, Source w, const long long* __restrict__ target, long long ignore, float* __restrict__ maxima) {
    const Source s = blockIdx.y ? w : h;
    float m = 0.f;
    for (long long r = blockIdx.x; r < s.rows; r += kMaxima) {
        if (blockIdx.y == 0 && target[r] == ignore) continue;
        const float* p = (const float*)s.p + r * s.ld;
        for (int c = threadIdx.x; c < s.cols; c += 256) {
            const float v = fabsf(p[c]);
            m = v <= 3.4028235e38f ? fmaxf(m, v) : m;
        }
    }
    __shared__ float red[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) maxima[blockIdx.y * kMaxima + blockIdx.x] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}
// the power of two that brings the largest magnitude to [2^14, 2^15)
__global__ __launch_bounds__(256) void exponents_kernel(const float* __restrict__ maxima, Scalars* __restrict__ sc) {
    __shared__ float red[2][4];
    for (int q = 0; q < 2; ++q) {
        float m = maxima[q * kMaxima + threadIdx.x];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        if ((threadIdx.x & 63) == 0) red[q][threadIdx.x >> 6] = m;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        const float* r = red[threadIdx.x];
        const float m = fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3]));
        const int e = m > 0.f ? 14 - ilogbf(m) : 0;
        if (threadIdx.x == 0) sc->eh = e; else sc->ew = e;
    }
}

template <int PL> __device__ __forceinline__ float logit_factor(const Scalars* sc, float scale) {
    if constexpr (PL == TWO) return ldexpf(scale, -(sc->eh + sc->ew));
    else return scale;
}

// ---- forward: maximum and sum of exponentials of each row of a tile of z, and the target's z.  partial [tile column][N]
template <class TileT>
__global__ __launch_bounds__(TileT::THREADS, TileT::THREADS == 512 ? 2 : 1) void lce_forward_kernel(Operand H, Operand W, int width, const Scalars* __restrict__ sc, float scale,
                                                                                                    const long long* __restrict__ target, float2* __restrict__ partial, float* __restrict__ ztarget) {
    UNFLOW_DYNAMIC_LDS(char, lds);
    const int mt = ceil_div(H.rows, TileT::BM), nt = ceil_div(W.rows, TileT::BN);
    int tm, tn;
    tile_of(xcd_remap((int)blockIdx.x, (int)gridDim.x), mt, nt, tm, tn);
    const int m0 = tm * TileT::BM, n0 = tn * TileT::BN;
    TileT T;
    T.run(H, W, 0, width, m0, n0, lds);
    const float f = logit_factor<TileT::PL>(sc, scale);
    float2* rows = reinterpret_cast<float2*>(lds);                                       // [WN][BM]
    const int wn = TileT::wave() % TileT::WN, group = ((int)threadIdx.x & 63) >> 4;
#pragma unroll
    for (int i = 0; i < TileT::MI; ++i) {
        const int m = m0 + TileT::row(i);
        const long long t = m < H.rows ? target[m] : -1;
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < TileT::NI; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int n = n0 + TileT::col(j) + r;
                const float z = n < W.rows ? T.acc[i][j][r] * f : -INFINITY;
                T.acc[i][j][r] = z;
                if (n == t && n < W.rows) ztarget[m] = z;
                top = fmaxf(top, z);
            }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < TileT::NI; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) sum += __expf(T.acc[i][j][r] - base);
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
            if (v.x != -INFINITY) sum += v.y * __expf(v.x - top);
            else sum += v.y;                                                              // (0, or NaN from a row of NaN, which fmaxf passes over)
        }
        partial[(long long)tn * H.rows + m0 + r] = make_float2(top, sum);
    }
}

// the tiles' (maximum, sum) pairs of a row joined in fixed order: 16 rows x 16 shares of the tiles per workgroup
__global__ __launch_bounds__(256) void lce_join_kernel(const float2* __restrict__ partial, int tiles, int N, int V, const long long* __restrict__ target, long long ignore,
                                                       const float* __restrict__ ztarget, float* __restrict__ lse, float* __restrict__ losses) {
    __shared__ float2 part[16][17];
    const int r = threadIdx.x & 15, share = threadIdx.x >> 4, m = blockIdx.x * 16 + r;
    float top = -INFINITY, sum = 0.f;
    if (m < N)
        for (int t = share; t < tiles; t += 16) {
            const float2 v = partial[(long long)t * N + m];
            const float both = fmaxf(top, v.x);
            const float base = both == -INFINITY ? 0.f : both;
            sum = sum * (top == -INFINITY ? 1.f : __expf(top - base)) + v.y * (v.x == -INFINITY ? 1.f : __expf(v.x - base));
            top = both;
        }
    part[share][r] = make_float2(top, sum);
    __syncthreads();
    if (share == 0 && m < N) {
        top = -INFINITY;
        for (int q = 0; q < 16; ++q) top = fmaxf(top, part[q][r].x);
        const float base = top == -INFINITY ? 0.f : top;
        sum = 0.f;
        for (int q = 0; q < 16; ++q) sum += part[q][r].y * (part[q][r].x == -INFINITY ? 1.f : expf(part[q][r].x - base));
        const float l = base + logf(sum);
        const long long t = target[m];
        lse[m] = l;
        losses[m] = t == ignore ? 0.f : (t >= 0 && t < V) ? l - ztarget[m] : NAN;
    }
}

// loss = sum of the rows' losses (mean: divided by the number of rows that are not ignored, at least 1), one workgroup, fixed order
__global__ __launch_bounds__(1024) void lce_reduce_kernel(const float* __restrict__ losses, const long long* __restrict__ target, long long ignore, int N, int mean, float* __restrict__ loss) {
    __shared__ float red[16], cnt[16];
    float s = 0.f, c = 0.f;
    for (int i = threadIdx.x; i < N; i += 1024) {
        s += losses[i];
        c += target[i] != ignore ? 1.f : 0.f;
    }
    s = wave_sum(s);
    c = wave_sum(c);
    if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = s; cnt[threadIdx.x >> 6] = c; }
    __syncthreads();
    if (threadIdx.x == 0) {
        s = c = 0.f;
        for (int q = 0; q < 16; ++q) { s += red[q]; c += cnt[q]; }
        loss[0] = mean ? s / fmaxf(c, 1.f) : s;
    }
}

// ---- backward
// uniform factors and the rows' weights: gscale[m] = upstream gradient of the row (1 where the loss is reduced; 0 where the row is ignored),
// one workgroup
__global__ __launch_bounds__(1024) void lce_weights_kernel(const float* __restrict__ gout, int reduction, float scale, const long long* __restrict__ target, long long ignore, int N,
                                                           int exponents, Scalars* __restrict__ sc, float* __restrict__ weight) {
    __shared__ float red[16], cnt[16];
    float top = 0.f, c = 0.f;
    for (int i = threadIdx.x; i < N; i += 1024) {
        const bool used = target[i] != ignore;
        const float g = used ? (reduction == 0 ? gout[i] : 1.f) : 0.f;
        weight[i] = g;
        const float a = fabsf(g);
        top = a <= 3.4028235e38f ? fmaxf(top, a) : top;
        c += used ? 1.f : 0.f;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    c = wave_sum(c);
    if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = top; cnt[threadIdx.x >> 6] = c; }
    __syncthreads();
    if (threadIdx.x == 0) {
        top = c = 0.f;
        for (int q = 0; q < 16; ++q) { top = fmaxf(top, red[q]); c += cnt[q]; }
        sc->gmax = top > 0.f ? top : 1.f;
        if (!exponents) sc->eh = sc->ew = 0;
        sc->factor = reduction == 0 ? scale : reduction == 1 ? scale * gout[0] / fmaxf(c, 1.f) : scale * gout[0];
    }
}

// fp16 planes hold probabilities times 2^14: 11 (22) bits of every probability down to 2^-28 (2^-17)
template <int EL> __host__ __device__ constexpr int probability_exponent() { return EL == FP16 ? 14 : 0; }

// a piece of G and of its transpose: classes [v0, v0 + vp).  G [N][packed vp] holds p - [v = t] (0 where the row is ignored), GT [vp][packed N] the
// same times the row's weight / gmax; columns behind N and vp up to the packed width are zero
template <class TileT>
__global__ __launch_bounds__(TileT::THREADS, TileT::THREADS == 512 ? 2 : 1) void lce_gradient_kernel(Operand H, Operand W, int width, const Scalars* __restrict__ sc, float scale,
                                                                                                     const long long* __restrict__ target, const float* __restrict__ lse, const float* __restrict__ weight,
                                                                                                     long long ignore, int v0, int vp, int V, u16* __restrict__ G, long long ldg, u16* __restrict__ GT, long long ldgt) {
    constexpr int PL = TileT::PL, EL = TileT::EL;
    UNFLOW_DYNAMIC_LDS(char, lds);
    const int mt = ceil_div(H.rows, TileT::BM), nt = ceil_div(vp, TileT::BN);
    int tm, tn;
    tile_of(xcd_remap((int)blockIdx.x, (int)gridDim.x), mt, nt, tm, tn);
    const int m0 = tm * TileT::BM, n0 = tn * TileT::BN;
    TileT T;
    const Operand piece{W.p + (long long)v0 * W.ld, W.ld, vp};
    T.run(H, piece, 0, width, m0, n0, lds);
    const float f = logit_factor<TileT::PL>(sc, scale), unit = (float)(1 << probability_exponent<EL>()), inv = 1.f / sc->gmax;
    const int wide_n = PL == TWO ? (int)round_up(vp, 32) : (int)round_up(vp, 8), wide_m = PL == TWO ? (int)round_up(H.rows, 32) : (int)round_up(H.rows, 8);
#pragma unroll
    for (int i = 0; i < TileT::MI; ++i) {
        const int m = m0 + TileT::row(i);
        const bool there = m < H.rows;
        const long long t = there ? target[m] : ignore;
        const bool used = t != ignore, known = t >= 0 && t < V;
        const float l = there ? lse[m] : 0.f, wgt = there ? weight[m] * inv : 0.f;
#pragma unroll
        for (int j = 0; j < TileT::NI; ++j) {
            const int n = n0 + TileT::col(j);
            f32x4 g;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float p = __expf(T.acc[i][j][r] * f - l);
                if (v0 + n + r == t) p -= 1.f;
                p = used ? (known ? p : NAN) : 0.f;
                g[r] = n + r < vp ? p * unit : 0.f;
            }
            if (there && n < wide_n) pack4<PL, EL>(G + (long long)m * ldg, n, g);
            if (m < wide_m) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n + r < vp) pack1<PL, EL>(GT + (long long)(n + r) * ldgt, m, used ? g[r] * wgt : 0.f);
            }
        }
    }
}

// C = A B^T over share `s` of `shares` of the packed width, added to (or, with `first`, stored in) fp32 sums [shares][rows of A][ldc]
template <class TileT>
__global__ __launch_bounds__(TileT::THREADS, TileT::THREADS == 512 ? 2 : 1) void gather_product_kernel(Operand A, Operand B, int width, int shares, float* __restrict__ C, long long ldc, int first) {
    UNFLOW_DYNAMIC_LDS(char, lds);
    const int mt = ceil_div(A.rows, TileT::BM), nt = ceil_div(B.rows, TileT::BN);
    const int id = xcd_remap((int)blockIdx.x, (int)gridDim.x), share = id / (mt * nt);
    int tm, tn;
    tile_of(id % (mt * nt), mt, nt, tm, tn);
    const int m0 = tm * TileT::BM, n0 = tn * TileT::BN;
    const int stages = ceil_div(width, 64), per = ceil_div(stages, shares);
    const int k0 = share * per * 64, k1 = (share + 1) * per * 64 < width ? (share + 1) * per * 64 : width;
    TileT T;
    T.run(A, B, k0, k1, m0, n0, lds);
    C += (long long)share * A.rows * ldc;
#pragma unroll
    for (int i = 0; i < TileT::MI; ++i) {
        const int m = m0 + TileT::row(i);
        if (m >= A.rows) continue;
        float* row = C + (long long)m * ldc;
        if (!first) {                                                  // (all of a row's loads before its sums: one wait, not one per load)
            f32x4 old[TileT::NI];
#pragma unroll
            for (int j = 0; j < TileT::NI; ++j) old[j] = n0 + TileT::col(j) < ldc ? *reinterpret_cast<const f32x4*>(row + n0 + TileT::col(j)) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < TileT::NI; ++j) T.acc[i][j] += old[j];
        }
#pragma unroll
        for (int j = 0; j < TileT::NI; ++j)
            if (n0 + TileT::col(j) < ldc) *reinterpret_cast<f32x4*>(row + n0 + TileT::col(j)) = T.acc[i][j];          // (ldc: the columns rounded up to 4)
    }
}

// C = A B^T times the uniform factor, in the gradient's type
template <class TileT, class T_>
__global__ __launch_bounds__(TileT::THREADS, TileT::THREADS == 512 ? 2 : 1) void weight_product_kernel(Operand A, Operand B, int width, const Scalars* __restrict__ sc, T_* __restrict__ C, long long ldc) {
    UNFLOW_DYNAMIC_LDS(char, lds);
    const int mt = ceil_div(A.rows, TileT::BM), nt = ceil_div(B.rows, TileT::BN);
    int tm, tn;
    tile_of(xcd_remap((int)blockIdx.x, (int)gridDim.x), mt, nt, tm, tn);
    const int m0 = tm * TileT::BM, n0 = tn * TileT::BN;
    TileT T;
    T.run(A, B, 0, width, m0, n0, lds);
    const float f = ldexpf(sc->factor * sc->gmax, -sc->eh - probability_exponent<TileT::EL>());
#pragma unroll
    for (int i = 0; i < TileT::MI; ++i)
#pragma unroll
        for (int j = 0; j < TileT::NI; ++j) {
            const int m = m0 + TileT::row(i), n = n0 + TileT::col(j), left = B.rows - n;
            if (m < A.rows && left > 0) store4<T_>(C + (long long)m * ldc + n, T.acc[i][j] * f, left < 4 ? left : 4);
        }
}

// gradient = (sum of the shares, in order) * uniform factor * (the row's weight), in the gradient's type
template <class T_>
__global__ __launch_bounds__(256) void finish_kernel(const float* __restrict__ C, long long ldc, int shares, int rows, int cols, const Scalars* __restrict__ sc, int by_h, int unit_exponent,
                                                     const float* __restrict__ weight, T_* __restrict__ out, long long ldo) {
    const float f = ldexpf(sc->factor * (weight ? 1.f : sc->gmax), -(by_h ? sc->eh : sc->ew) - unit_exponent);
    const long long per = ldc / 4, total = per * rows;
    for (long long g = blockIdx.x * 256ll + threadIdx.x; g < total; g += gridDim.x * 256ll) {
        const long long r = g / per;
        const int n = (int)(g - r * per) * 4;
        f32x4 v = *reinterpret_cast<const f32x4*>(C + r * ldc + n);
        for (int s = 1; s < shares; ++s) v += *reinterpret_cast<const f32x4*>(C + ((long long)s * rows + r) * ldc + n);
        v *= weight ? f * weight[r] : f;
        store4<T_>(out + r * ldo + n, v, cols - n < 4 ? cols - n : 4);
    }
}

// ---- the host side
using T256b = Tile<256, 256, 2, 4, ONE, BF16>;
using T128b = Tile<128, 128, 2, 2, ONE, BF16>;
using T64b = Tile<64, 64, 2, 2, ONE, BF16>;
using T256h = Tile<256, 256, 2, 4, ONE, FP16>;
using T128h = Tile<128, 128, 2, 2, ONE, FP16>;
using T64h = Tile<64, 64, 2, 2, ONE, FP16>;
using T256t = Tile<256, 256, 2, 4, TWO, FP16>;
using T128t = Tile<128, 128, 2, 2, TWO, FP16>;
using T64t = Tile<64, 64, 2, 2, TWO, FP16>;

static int tiles(long long m, long long n, int size) { return (int)(((m + size - 1) / size) * ((n + size - 1) / size)); }
// The largest tile that still gives every CU one (256 of them): a tile of twice the side reads half as much per product.  Below that the chip
// is not full and the smaller tile wins.
static int tile_size(long long m, long long n) { return tiles(m, n, 256) >= 224 ? 256 : tiles(m, n, 128) >= 224 ? 128 : 64; }

#define WITH_TILE(planes, el, size, ...)                                                                                      \
    do {                                                                                                                      \
        if (planes == TWO) { if (size == 256) { using TileT = T256t; __VA_ARGS__; } else if (size == 128) { using TileT = T128t; __VA_ARGS__; } else { using TileT = T64t; __VA_ARGS__; } } \
        else if (el == FP16) { if (size == 256) { using TileT = T256h; __VA_ARGS__; } else if (size == 128) { using TileT = T128h; __VA_ARGS__; } else { using TileT = T64h; __VA_ARGS__; } } \
        else { if (size == 256) { using TileT = T256b; __VA_ARGS__; } else if (size == 128) { using TileT = T128b; __VA_ARGS__; } else { using TileT = T64b; __VA_ARGS__; } }                   \
    } while (0)

#define LAUNCH_TILES(kernel, count, ...)                                                                                      \
    do {                                                                                                                      \
        if (TileT::LDS > 65536) (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, TileT::LDS); \
        UNFLOW_LAUNCH(kernel, dim3(count), dim3(TileT::THREADS), TileT::LDS, stream, __VA_ARGS__);                            \
    } while (0)

// What a call needs of its workspace, and where.
struct Plan {
    int planes, el;
    bool pack_h, pack_w;                 // the inputs are not operands as they are
    long long wd, wn;                    // packed width of D and of N
    int size_z;                          // tile of the logits
    // forward
    long long scalars, maxima, hp, wp, partial, ztarget, losses, forward_bytes;
    // backward
    int vp, size_g, size_h, size_w, shares_h, shares_w;
    long long wvp, ldh_sum, ldw_sum;
    long long weight, ht, wt, g, gt, sum_h, sum_w, backward_bytes;
};

static bool as_is(const void* p, long long ld, int D, int dtype) { return dtype != kFp32 && D % 8 == 0 && ld % 8 == 0 && ((size_t)p & 15) == 0; }

// Products whose tiles do not fill the chip are cut along what they sum over, into at most 16 shares of at least 8 stages.
static int shares_of(long long m, long long n, int size, long long width) {
    const long long stages = (width + 63) / 64;
    long long want = 256 / tiles(m, n, size);
    if (want > stages / 8) want = stages / 8;
    if (want > 16) want = 16;
    if (want <= 1) return 1;
    const long long per = (stages + want - 1) / want;          // (no share is empty)
    return (int)((stages + per - 1) / per);
}

static Plan plan_of(const void* h, long long ldh, const void* w, long long ldw, int N, int V, int D, int dtype, bool need_h, bool need_w) {
    Plan p{};
    p.planes = dtype == kFp32 ? TWO : ONE;
    p.el = dtype == kBf16 ? BF16 : FP16;
    p.pack_h = !as_is(h, ldh, D, dtype);
    p.pack_w = !as_is(w, ldw, D, dtype);
    p.wd = packed_width(p.planes, D);
    p.wn = packed_width(p.planes, N);
    long long at = 0;
    auto take = [&](long long bytes) { const long long a = at; at += round_up(bytes, 256); return a; };
    p.scalars = take(sizeof(Scalars));
    p.maxima = take(2 * kMaxima * 4);
    p.hp = p.pack_h ? take(2 * p.wd * N) : 0;
    p.wp = p.pack_w ? take(2 * p.wd * V) : 0;
    const long long common = at;
    p.size_z = tile_size(N, V);
    p.partial = take(8ll * ceil_div(V, p.size_z) * N);
    p.ztarget = take(4ll * N);
    p.losses = take(4ll * N);
    p.forward_bytes = at;
    at = common;
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
    p.size_g = tile_size(N, p.vp);
    p.size_h = tile_size(N, D);
    p.size_w = tile_size(p.vp, D);
    p.shares_h = shares_of(N, D, p.size_h, p.wvp);
    p.shares_w = shares_of(p.vp, D, p.size_w, p.wn);
    p.weight = take(4ll * N);
    p.g = take(2 * p.wvp * N);
    p.gt = take(2 * p.wn * p.vp);
    p.ldh_sum = round_up(D, 4);
    if (need_h) {
        p.wt = take(2 * p.wvp * D);
        p.sum_h = take(4ll * p.shares_h * p.ldh_sum * N);
    }
    if (need_w) {
        p.ht = take(2 * p.wn * D);
        if (p.shares_w > 1) p.sum_w = take(4ll * p.shares_w * p.ldh_sum * p.vp);
    }
    p.backward_bytes = at;
    return p;
}

static int blocks_for(long long work) { const long long b = (work + 255) / 256; return (int)(b < 1 ? 1 : b > 8192 ? 8192 : b); }

template <int PL, int EL, class T>
static void pack_rows(const Source& s, u16* dst, long long ldd, hipStream_t stream) {
    const int width = (int)(PL == TWO ? ldd / 2 : ldd);
    UNFLOW_LAUNCH((pack_rows_kernel<T, PL, EL>), dim3(blocks_for((long long)s.rows * (width / 4))), dim3(256), 0, stream, s, dst, ldd, width);
}
template <int PL, int EL, class T>
static void pack_columns(const Source& s, u16* dst, long long ldd, hipStream_t stream) {
    const int width = (int)(PL == TWO ? ldd / 2 : ldd);
    UNFLOW_LAUNCH((pack_columns_kernel<T, PL, EL>), dim3(ceil_div(width, 64), ceil_div(s.cols, 64)), dim3(256), 0, stream, s, dst, ldd, width);
}
static void pack_rows_of(int dtype, const Source& s, u16* dst, long long ldd, hipStream_t stream) {
    if (dtype == kFp32) pack_rows<TWO, FP16, float>(s, dst, ldd, stream);
    else if (dtype == kBf16) pack_rows<ONE, BF16, __bf16>(s, dst, ldd, stream);
    else pack_rows<ONE, FP16, _Float16>(s, dst, ldd, stream);
}
static void pack_columns_of(int dtype, const Source& s, u16* dst, long long ldd, hipStream_t stream) {
    if (dtype == kFp32) pack_columns<TWO, FP16, float>(s, dst, ldd, stream);
    else if (dtype == kBf16) pack_columns<ONE, BF16, __bf16>(s, dst, ldd, stream);
    else pack_columns<ONE, FP16, _Float16>(s, dst, ldd, stream);
}

// H and W as operands (packed into the workspace where they are none by themselves), and the exponents they were packed with
static void operands(const Plan& p, const void* h, long long ldh, const void* w, long long ldw, const long long* target, long long ignore, int N, int V, int D, int dtype, char* ws, hipStream_t stream,
                     Operand& H, Operand& W) {
    Scalars* sc = (Scalars*)(ws + p.scalars);
    const int *eh = nullptr, *ew = nullptr;
    if (dtype == kFp32) {
        UNFLOW_LAUNCH(largest_kernel, dim3(kMaxima, 2), dim3(256), 0, stream, Source{h, ldh, N, D, nullptr}, Source{w, ldw, V, D, nullptr}, target, ignore, (float*)(ws + p.maxima));
        UNFLOW_LAUNCH(exponents_kernel, dim3(1), dim3(256), 0, stream, (const float*)(ws + p.maxima), sc);
        eh = &sc->eh;
        ew = &sc->ew;
    }
    H = Operand{(const u16*)h, ldh, N};
    W = Operand{(const u16*)w, ldw, V};
    if (p.pack_h) {
        H = Operand{(const u16*)(ws + p.hp), p.wd, N};
        pack_rows_of(dtype, Source{h, ldh, N, D, eh}, (u16*)(ws + p.hp), p.wd, stream);
    }
    if (p.pack_w) {
        W = Operand{(const u16*)(ws + p.wp), p.wd, V};
        pack_rows_of(dtype, Source{w, ldw, V, D, ew}, (u16*)(ws + p.wp), p.wd, stream);
    }
}

static bool sizes_ok(long long ldh, long long ldw, int N, int V, int D, int dtype, int reduction) {
    return N > 0 && V > 0 && D > 0 && N <= UNFLOW_LCE_MAX_ROWS && D <= UNFLOW_LCE_MAX_DIM && ldh >= D && ldw >= D && ldh <= UNFLOW_LCE_MAX_DIM && ldw <= UNFLOW_LCE_MAX_DIM &&
           dtype >= kFp32 && dtype <= kFp16 && reduction >= 0 && reduction <= 2;
}

}  // namespace

extern "C" int unflow_linear_ce_workspace(const void* hidden, long long ldh, const void* weight, long long ldw, int N, int V, int D, int dtype, int need_h, int need_w,
                                          long long* forward_bytes, long long* backward_bytes) {
    UNFLOW_REQUIRE(forward_bytes && backward_bytes && sizes_ok(ldh, ldw, N, V, D, dtype, 0));
    const Plan p = plan_of(hidden, ldh, weight, ldw, N, V, D, dtype, need_h != 0, need_w != 0);
    *forward_bytes = p.forward_bytes;
    *backward_bytes = p.backward_bytes;
    return 0;
}

extern "C" int unflow_linear_ce_fwd(const void* hidden, long long ldh, const void* weight, long long ldw, const long long* target, int N, int V, int D, int dtype, float scale,
                                    long long ignore_index, int reduction, float* loss, float* lse, void* workspace, long long workspace_bytes, void* stream_) {
    UNFLOW_REQUIRE(hidden && weight && target && loss && lse && workspace && sizes_ok(ldh, ldw, N, V, D, dtype, reduction));
    const Plan p = plan_of(hidden, ldh, weight, ldw, N, V, D, dtype, false, false);
    UNFLOW_REQUIRE(workspace_bytes >= p.forward_bytes);
    hipStream_t stream = (hipStream_t)stream_;
    char* ws = (char*)workspace;
    Operand H, W;
    operands(p, hidden, ldh, weight, ldw, target, ignore_index, N, V, D, dtype, ws, stream, H, W);
    const Scalars* sc = (const Scalars*)(ws + p.scalars);
    const int width = (int)(p.planes == TWO ? p.wd : D + (8 - D % 8) % 8);
    const int count = tiles(N, V, p.size_z);
    float2* partial = (float2*)(ws + p.partial);
    float* zt = (float*)(ws + p.ztarget);
    WITH_TILE(p.planes, p.el, p.size_z, LAUNCH_TILES((lce_forward_kernel<TileT>), count, H, W, width, sc, scale, target, partial, zt));
    float* losses = reduction == 0 ? loss : (float*)(ws + p.losses);
    UNFLOW_LAUNCH(lce_join_kernel, dim3(ceil_div(N, 16)), dim3(256), 0, stream, (const float2*)partial, ceil_div(V, p.size_z), N, V, target, ignore_index, (const float*)zt, lse, losses);
    if (reduction != 0) UNFLOW_LAUNCH(lce_reduce_kernel, dim3(1), dim3(1024), 0, stream, (const float*)losses, target, ignore_index, N, reduction == 1 ? 1 : 0, loss);
    return unflow_launch_status();
}

extern "C" int unflow_linear_ce_bwd(const void* hidden, long long ldh, const void* weight, long long ldw, const long long* target, const float* lse, const float* gout, int N, int V, int D,
                                    int dtype, float scale, long long ignore_index, int reduction, void* dhidden, void* dweight, void* workspace, long long workspace_bytes, void* stream_) {
    UNFLOW_REQUIRE(hidden && weight && target && lse && gout && (dhidden || dweight) && workspace && sizes_ok(ldh, ldw, N, V, D, dtype, reduction));
    const Plan p = plan_of(hidden, ldh, weight, ldw, N, V, D, dtype, dhidden != nullptr, dweight != nullptr);
    UNFLOW_REQUIRE(workspace_bytes >= p.backward_bytes);
    hipStream_t stream = (hipStream_t)stream_;
    char* ws = (char*)workspace;
    Operand H, W;
    operands(p, hidden, ldh, weight, ldw, target, ignore_index, N, V, D, dtype, ws, stream, H, W);
    Scalars* sc = (Scalars*)(ws + p.scalars);
    const int width = (int)(p.planes == TWO ? p.wd : D + (8 - D % 8) % 8);
    const int unit = p.el == FP16 ? probability_exponent<FP16>() : probability_exponent<BF16>();
    const long long esize = dtype == kFp32 ? 4 : 2;
    float* rows = (float*)(ws + p.weight);
    UNFLOW_LAUNCH(lce_weights_kernel, dim3(1), dim3(1024), 0, stream, gout, reduction, scale, target, ignore_index, N, dtype == kFp32 ? 1 : 0, sc, rows);
    const int* eh = dtype == kFp32 ? &sc->eh : nullptr;
    const int* ew = dtype == kFp32 ? &sc->ew : nullptr;
    u16 *G = (u16*)(ws + p.g), *GT = (u16*)(ws + p.gt);
    const Operand HT{(const u16*)(ws + p.ht), p.wn, D};
    if (dweight) pack_columns_of(dtype, Source{hidden, ldh, N, D, eh, target, ignore_index}, (u16*)(ws + p.ht), p.wn, stream);
    for (int v0 = 0; v0 < V; v0 += p.vp) {
        const int vp = V - v0 < p.vp ? V - v0 : p.vp;
        const long long wvp = packed_width(p.planes, vp);
        const int count_g = tiles(N, vp, p.size_g);
        WITH_TILE(p.planes, p.el, p.size_g, LAUNCH_TILES((lce_gradient_kernel<TileT>), count_g, H, W, width, (const Scalars*)sc, scale, target, lse, (const float*)rows, ignore_index, v0, vp, V, G, p.wvp, GT, p.wn));
        if (dhidden) {
            pack_columns_of(dtype, Source{(const char*)weight + v0 * ldw * esize, ldw, vp, D, ew}, (u16*)(ws + p.wt), wvp, stream);
            const Operand A{G, p.wvp, N}, B{(const u16*)(ws + p.wt), wvp, D};
            float* sums = (float*)(ws + p.sum_h);
            const int count = tiles(N, D, p.size_h) * p.shares_h;
            WITH_TILE(p.planes, p.el, p.size_h, LAUNCH_TILES((gather_product_kernel<TileT>), count, A, B, (int)wvp, p.shares_h, sums, p.ldh_sum, v0 == 0 ? 1 : 0));
        }
        if (dweight) {
            const Operand A{GT, p.wn, vp};
            char* out = (char*)dweight + (long long)v0 * D * esize;
            if (p.shares_w > 1) {
                float* sums = (float*)(ws + p.sum_w);
                const int count = tiles(vp, D, p.size_w) * p.shares_w;
                WITH_TILE(p.planes, p.el, p.size_w, LAUNCH_TILES((gather_product_kernel<TileT>), count, A, HT, (int)p.wn, p.shares_w, sums, p.ldh_sum, 1));
                const int blocks = blocks_for((long long)vp * (p.ldh_sum / 4));
                if (dtype == kFp32) UNFLOW_LAUNCH((finish_kernel<float>), dim3(blocks), dim3(256), 0, stream, (const float*)sums, p.ldh_sum, p.shares_w, vp, D, (const Scalars*)sc, 1, unit, (const float*)nullptr, (float*)out, (long long)D);
                else if (dtype == kBf16) UNFLOW_LAUNCH((finish_kernel<__bf16>), dim3(blocks), dim3(256), 0, stream, (const float*)sums, p.ldh_sum, p.shares_w, vp, D, (const Scalars*)sc, 1, unit, (const float*)nullptr, (__bf16*)out, (long long)D);
                else UNFLOW_LAUNCH((finish_kernel<_Float16>), dim3(blocks), dim3(256), 0, stream, (const float*)sums, p.ldh_sum, p.shares_w, vp, D, (const Scalars*)sc, 1, unit, (const float*)nullptr, (_Float16*)out, (long long)D);
            } else {
                const int count = tiles(vp, D, p.size_w);
                if (p.planes == TWO) WITH_TILE(TWO, FP16, p.size_w, LAUNCH_TILES((weight_product_kernel<TileT, float>), count, A, HT, (int)p.wn, (const Scalars*)sc, (float*)out, (long long)D));
                else if (p.el == FP16) WITH_TILE(ONE, FP16, p.size_w, LAUNCH_TILES((weight_product_kernel<TileT, _Float16>), count, A, HT, (int)p.wn, (const Scalars*)sc, (_Float16*)out, (long long)D));
                else WITH_TILE(ONE, BF16, p.size_w, LAUNCH_TILES((weight_product_kernel<TileT, __bf16>), count, A, HT, (int)p.wn, (const Scalars*)sc, (__bf16*)out, (long long)D));
            }
        }
    }
    if (dhidden) {
        const float* sums = (const float*)(ws + p.sum_h);
        const int blocks = blocks_for((long long)N * (p.ldh_sum / 4));
        if (dtype == kFp32) UNFLOW_LAUNCH((finish_kernel<float>), dim3(blocks), dim3(256), 0, stream, sums, p.ldh_sum, p.shares_h, N, D, (const Scalars*)sc, 0, unit, (const float*)rows, (float*)dhidden, (long long)D);
        else if (dtype == kBf16) UNFLOW_LAUNCH((finish_kernel<__bf16>), dim3(blocks), dim3(256), 0, stream, sums, p.ldh_sum, p.shares_h, N, D, (const Scalars*)sc, 0, unit, (const float*)rows, (__bf16*)dhidden, (long long)D);
        else UNFLOW_LAUNCH((finish_kernel<_Float16>), dim3(blocks), dim3(256), 0, stream, sums, p.ldh_sum, p.shares_h, N, D, (const Scalars*)sc, 0, unit, (const float*)rows, (_Float16*)dhidden, (long long)D);
    }
    return unflow_launch_status();
}
