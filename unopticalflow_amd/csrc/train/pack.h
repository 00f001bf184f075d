// Matrices of fp32 / bf16 / fp16 numbers into the packed operand rows of mfma16.h, as they are or transposed.  Both are one read and one write of
// the matrix; the transposed form goes through an LDS tile so that either side is contiguous.
#pragma once
#include "mfma16.h"

namespace {

// What is read: rows x cols, `ld` elements from row to row.  A row r with label[r] == skip does not count (label == nullptr: every row does).
struct Source { const void* p; long long ld; int rows, cols; const long long* label = nullptr; long long skip = 0; };

// the first n = 0 .. 4 of four numbers, zeros behind them
template <class T> __device__ __forceinline__ f32x4 load4(const T* p, int n) {
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

// dst row c = source column c times 2^e, for the `cols` columns; `width` >= rows numbers a dst row holds, zeros behind rows and for rows that do
// not count.  The 64 x 64 tile (bx, by) of ceil(width / 64) x ceil(cols / 64)
template <class T, int PL, int EL>
__device__ __forceinline__ void pack_columns_tile(const Source& s, int e, u16* __restrict__ dst, long long ldd, int width, int bx, int by) {
    __shared__ float tile[64][65];
    const int r0 = bx * 64, c0 = by * 64;
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
