// The 8-bit cache: how its blocks lie in memory, and the sequences of a call.
//
// A block holds 32 tokens of every KV head; a head's part of it is a unit: a header, the keys, the values, one byte each. A value is q * scale with
// an integer q of -127 .. 127 (the byte is q + 128) and a power of two as the scale of a unit's keys, another of its values: products with it are exact,
// a block whose scale grows is brought to it by shifting, and every program that follows the definition gets the same bits. (amax / 127 as the scale keeps
// half a bit more on average, and rounds what was there at every new largest value.)
//
// Bytes lie as mma.sync.m16n8k16 takes them (a lane's words side by side, no two lanes of a load in a bank):
//   keys   : tiles of eight keys; a lane (n = key of the tile, t) has dimensions t * HD / 4 .. of key n, 16 at a time;
//   values : 16 dimensions at a time; a lane (n = dimension of eight, t) has tokens 4 t .. 4 t + 3 and 16 + 4 t .. of dimensions n and 8 + n.
// Key n of tile j is the token that the probabilities of a lane belong to: 16 (j / 2) + 4 (n / 2) + 2 (j % 2) + n % 2.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "kernels.h"

namespace b2 {
namespace kv8 {

struct __align__(16) Header {
    float k_scale;   // 0: never written
    uint32_t k_bad;  // tokens whose keys had a value that is not finite: they count as NaN
    float v_scale;
    uint32_t v_bad;
    uint32_t pad[4];
};
static_assert(sizeof(Header) == KV8_HEADER);

__host__ __device__ constexpr uint32_t unit_bytes(uint32_t hd) { return KV8_HEADER + 2 * KV8_BLOCK * hd; }

// Offset of token `tok` (of 32), dimension d, in the keys and in the values of a unit.
template <int HD>
__device__ __forceinline__ uint32_t key_at(uint32_t tok, uint32_t d) {
    constexpr uint32_t QD = HD / 4;
    const uint32_t j = 2 * (tok >> 4) + ((tok >> 1) & 1), n = 2 * ((tok & 15) >> 2) + (tok & 1), r = d % QD;
    return j * (8 * HD) + (r >> 4) * 512 + (n * 4 + d / QD) * 16 + (r & 15);
}
__device__ __forceinline__ uint32_t value_at(uint32_t tok, uint32_t d) {
    return (d >> 4) * 512 + ((d & 7) * 4 + ((tok & 15) >> 2)) * 16 + ((d >> 3) & 1) * 8 + (tok >> 4) * 4 + (tok & 3);
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// The sequence's rows in the arrays of the call (r0, count) and its first position. False, with the status word set, where they lie outside what the
// host said; nothing of such a sequence is read or written.
struct Seq {
    uint32_t r0, count, start;
};
__device__ __forceinline__ bool sequence(const Kv8Seqs& c, uint32_t s, Seq* out, uint32_t* status) {
    long long r0, r1;
    if (c.rows) {
        r0 = c.rows[s];
        r1 = c.rows[s + 1];
    } else {
        r0 = (long long)s * c.max_rows;
        r1 = r0 + c.max_rows;
    }
    const long long start = c.start[s];
    if (r0 < 0 || r1 < r0 || r1 > (long long)c.n_rows || start < 0 || start + (r1 - r0) > (long long)c.max_blocks * KV8_BLOCK) {
        *(volatile uint32_t*)status = KV8_BAD_SEQUENCE;
        return false;
    }
    out->r0 = (uint32_t)r0;
    out->count = (uint32_t)(r1 - r0);
    out->start = (uint32_t)start;
    return true;
}
// The cache's number of the sequence's block b < max_blocks; -1, with the status word set, where the table names one that the cache does not have.
__device__ __forceinline__ int block_of(const Kv8Cache& k, const Kv8Seqs& c, uint32_t s, uint32_t b, uint32_t* status) {
    const long long at = (long long)s * c.max_blocks + b;
    const long long id = c.table ? (long long)c.table[at] : at;
    if (id < 0 || id >= (long long)k.n_blocks) {
        *(volatile uint32_t*)status = KV8_BAD_BLOCK;
        return -1;
    }
    return (int)id;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// Four values; `aligned`: to 16 bytes (f32) or 8.
__device__ __forceinline__ void load4(float (&v)[4], const float* p, bool aligned) {
    if (aligned) {
        const float4 x = *(const float4*)p;
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = p[i];
    }
}
template <typename T>
__device__ __forceinline__ void load4(float (&v)[4], const T* p, bool aligned) {
    if (aligned) {
        const uint2 x = *(const uint2*)p;
        alignas(8) T t[4];
        *(uint2*)t = x;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = to_f32<T>(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = to_f32<T>(p[i]);
    }
}

// Two f32 operations an instruction, and the largest of three.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

}  // namespace kv8
}  // namespace b2
