// Matrices of fp32 / bf16 / fp16 numbers into the packed operand rows of mfma16.h, as they are or transposed.  Both are one read and one write of
// the matrix; the transposed form goes through an LDS tile so that either side is contiguous.
#pragma once
#include "mfma16.h"

namespace {

// What is read: rows x cols, `ld` elements from row to row.  Numbers are multiplied by 2^*exp (exp == nullptr: as they are).  A row r with
// label[r] == skip counts as zeros (pack_columns; label == nullptr: none does).
struct Source { const void* p; long long ld; int rows, cols; const int* exp; const long long* label = nullptr; long long skip = 0; };

template <class T> __device__ __forceinline__ f32x4 load4(const T* p, int n) {               // the first n = 0 .. 4 of four numbers, zeros behind them
    f32x4 v{0.f, 0.f, 0.f, 0.f};
    if (n >= 4 && ((size_t)p & (4 * sizeof(T) - 1)) == 0) {
        if constexpr (sizeof(T) == 4) return *reinterpret_cast<const f32x4*>(p);
        else {
            const u32x2 h = *reinterpret_cast<const u32x2*>(p);
            const u16 e[4] = {(u16)h[0], (u16)(h[0] >> 16), (u16)h[1], (u16)(h[1] >> 16)};
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = (float)__builtin_bit_cast(T, e[r]);
            return v;
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (r < n) v[r] = (float)p[r];
    return v;
}
__device__ __forceinline__ f32x4 scaled(f32x4 v, int e) { return f32x4{ldexpf(v[0], e), ldexpf(v[1], e), ldexpf(v[2], e), ldexpf(v[3], e)}; }

// dst row r = source row r; `width` (numbers a row holds, a multiple of 4: packed_width of ONE, half of it for TWO) >= cols, zeros behind cols
template <class T, int PL, int EL>
__global__ __launch_bounds__(256) void pack_rows_kernel(Source s, u16* __restrict__ dst, long long ldd, int width) {
    const int e = s.exp ? *s.exp : 0;
    const long long per = width / 4, total = per * s.rows;
    for (long long g = blockIdx.x * 256ll + threadIdx.x; g < total; g += gridDim.x * 256ll) {
        const long long r = g / per;
        const int k = (int)(g - r * per) * 4;
        pack4<PL, EL>(dst + r * ldd, k, scaled(load4((const T*)s.p + r * s.ld + k, s.cols - k), e));
    }
}

// dst row c = source column c, for the `cols` columns; `width` >= rows numbers a dst row holds, zeros behind rows.  64 x 64 tiles, grid
// (ceil(width / 64), ceil(cols / 64))
template <class T, int PL, int EL>
__global__ __launch_bounds__(256) void pack_columns_kernel(Source s, u16* __restrict__ dst, long long ldd, int width) {
    __shared__ float tile[64][65];
    const int e = s.exp ? *s.exp : 0;
    const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64;
    const int x = (threadIdx.x & 15) * 4, y = threadIdx.x >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = r0 + y + 16 * i, c = c0 + x;
        const bool there = r < s.rows && !(s.label && s.label[r] == s.skip);
        const f32x4 v = scaled(there ? load4((const T*)s.p + r * s.ld + c, s.cols - c) : f32x4{0.f, 0.f, 0.f, 0.f}, e);
#pragma unroll
        for (int k = 0; k < 4; ++k) tile[y + 16 * i][x + k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = c0 + y + 16 * i, r = r0 + x;
        if (c < s.cols && r < width) {
            f32x4 v;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = tile[x + k][y + 16 * i];
            pack4<PL, EL>(dst + (long long)c * ldd, r, v);
        }
    }
}

}  // namespace
