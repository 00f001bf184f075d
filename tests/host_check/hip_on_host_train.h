// What the training operators (csrc/train) name beyond hip_on_host.h, in host form (TEST INFRASTRUCTURE; force-included by
// tests/train_on_host.py): the wave ballot, the fp16 matrix instruction, and the conversions the compiler calls for.
#pragma once
#include "hip_on_host.h"

struct alignas(16) uint4 { unsigned x, y, z, w; };

namespace hip_on_host { inline unsigned long long ballots[16]; }
static inline unsigned long long __ballot(int p) {
    const unsigned wave = hip_on_host::lane_id >> 6;
    __syncthreads();
    hip_on_host::ballots[wave] = 0;
    __syncthreads();
    if (p) hip_on_host::ballots[wave] |= 1ull << (hip_on_host::lane_id & 63u);
    __syncthreads();
    return hip_on_host::ballots[wave];
}
static inline int hip_on_host_readlane(int v, int lane) {
    static int values[1024];
    __syncthreads();
    values[hip_on_host::lane_id] = v;
    __syncthreads();
    const int r = values[(hip_on_host::lane_id & ~63u) + (unsigned)lane];
    __syncthreads();
    return r;
}
#define __builtin_amdgcn_readlane(v, lane) hip_on_host_readlane(v, lane)
static inline int __popcll(unsigned long long v) { return __builtin_popcountll(v); }

// v_mfma_f32_16x16x32_f16: the lane layouts of the bf16 form (hip_on_host.h)
typedef _Float16 hip_on_host_f16x8 __attribute__((ext_vector_type(8)));
static inline hip_on_host_v4f hip_on_host_mfma_16x16x32_f16(hip_on_host_f16x8 a, hip_on_host_f16x8 b, hip_on_host_v4f c) {
    const unsigned me = hip_on_host::lane_id, wave0 = me & ~63u, l = me & 63u;
    static float fa[1024][8], fb[1024][8];
    for (int e = 0; e < 8; ++e) { fa[me][e] = (float)a[e]; fb[me][e] = (float)b[e]; }
    __syncthreads();
    hip_on_host_v4f d = c;
    const unsigned col = l & 15u;
    for (int reg = 0; reg < 4; ++reg) {
        const unsigned row = 4u * (l >> 4) + (unsigned)reg;
        float acc = c[reg];
        for (int k = 0; k < 32; ++k) acc += fa[wave0 + row + 16u * (unsigned)(k >> 3)][k & 7] * fb[wave0 + col + 16u * (unsigned)(k >> 3)][k & 7];
        d[reg] = acc;
    }
    __syncthreads();
    return d;
}
#define __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, x, y, z) hip_on_host_mfma_16x16x32_f16(a, b, c)

// the bf16 form for workgroups of up to 1024 lanes (hip_on_host.h holds 256)
static inline hip_on_host_v4f hip_on_host_mfma_16x16x32_bf16_wide(hip_on_host_bf16x8 a, hip_on_host_bf16x8 b, hip_on_host_v4f c) {
    const unsigned me = hip_on_host::lane_id, wave0 = me & ~63u, l = me & 63u;
    static float fa[1024][8], fb[1024][8];
    for (int e = 0; e < 8; ++e) { fa[me][e] = (float)a[e]; fb[me][e] = (float)b[e]; }
    __syncthreads();
    hip_on_host_v4f d = c;
    const unsigned col = l & 15u;
    for (int reg = 0; reg < 4; ++reg) {
        const unsigned row = 4u * (l >> 4) + (unsigned)reg;
        float acc = c[reg];
        for (int k = 0; k < 32; ++k) acc += fa[wave0 + row + 16u * (unsigned)(k >> 3)][k & 7] * fb[wave0 + col + 16u * (unsigned)(k >> 3)][k & 7];
        d[reg] = acc;
    }
    __syncthreads();
    return d;
}
#undef __builtin_amdgcn_mfma_f32_16x16x32_bf16
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, x, y, z) hip_on_host_mfma_16x16x32_bf16_wide(a, b, c)

extern "C" __attribute__((weak)) __bf16 __truncsfbf2(float f) {          // round to nearest even, NaN stays NaN
    unsigned u;
    memcpy(&u, &f, 4);
    unsigned short h = (unsigned short)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
    if ((u & 0x7fffffffu) > 0x7f800000u) h = (unsigned short)((u >> 16) | 0x40u);
    __bf16 r;
    memcpy(&r, &h, 2);
    return r;
}

// v_mfma_f32_16x16x4_f32: lane l holds row (column) l & 15, k = l >> 4
static inline hip_on_host_v4f hip_on_host_mfma_16x16x4_f32(float a, float b, hip_on_host_v4f c) {
    const unsigned me = hip_on_host::lane_id, wave0 = me & ~63u, l = me & 63u;
    static float fa[1024], fb[1024];
    fa[me] = a; fb[me] = b;
    __syncthreads();
    hip_on_host_v4f d = c;
    for (int reg = 0; reg < 4; ++reg)
        for (unsigned k = 0; k < 4; ++k) d[reg] += fa[wave0 + 4u * (l >> 4) + (unsigned)reg + 16u * k] * fb[wave0 + (l & 15u) + 16u * k];
    __syncthreads();
    return d;
}
#define __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, x, y, z) hip_on_host_mfma_16x16x4_f32(a, b, c)

#define __builtin_amdgcn_exp2f(v) exp2f(v)

// LDS-DMA through a byte range (device_forms.h): landed when the call returns
typedef hip_on_host::Rsrc byte_range;
static inline byte_range range_of(const void* p, int bytes) { return byte_range{(char*)p, (unsigned)bytes}; }
typedef char* lds_address;
static inline lds_address address_in_lds(char* p) { return p; }
static inline void copy16_to_lds(byte_range r, lds_address to, unsigned offset) { hip_on_host::buf_load<16>(r, (int)offset, 0, to + (hip_on_host::lane_id & 63u) * 16); }
