// Rows of logits before a token is chosen (the reference does this on the host, src/sampler.rs): for every token that the row's history has c > 0 times
//   l = l > 0 ? l / repeat : l * repeat,  l -= frequency c + presence,
// then a bias where the row's list has one (the last entry of a token counts), -inf where the mask does not allow it; and the first largest.
// Every operation is a rounding of f32 of its own, so the values are those of the same formulas anywhere; 16-bit rows are rounded once at the end, and
// the choice is among what is stored.
//
// A cluster of CTAs has a row, a slice of the tokens each; what the lists say of a slice's tokens is counted in shared memory (integers, so the order of the
// atomics does not matter), every list read once by each CTA. One pass over the logits, bound by their bytes, or for few rows by latency.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kernels.h"
#include "pdl.cuh"

namespace b2 {

namespace {

constexpr int LG_THREADS = 512, LG_PART = 8192;  // tokens that are counted at a time

struct LgArgs {
    const void* x;
    void* out;
    size_t x_stride, out_stride;
    uint32_t n, slice, part;
    LogitRulesDev r;
    int32_t* pick;
    uint32_t* status;
    int aligned;
};

template <typename T>
__device__ __forceinline__ float as_f32(T v) {
    if constexpr (std::is_same<T, float>::value) return v;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
    else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T rounded(float v) {
    if constexpr (std::is_same<T, float>::value) return v;
    else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
    else return __float2bfloat16_rn(v);
}
__device__ __forceinline__ uint32_t lg_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t lg_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void lg_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t lg_peer(const void* p, uint32_t cta) {
    uint32_t a, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(cta));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
// (a, i) against (b, j): the larger, of equals the lower index; what is not above -inf is nothing.
__device__ __forceinline__ void better(float& b, int& j, float a, int i) {
    if (a > b || (a == b && i < j && a > -INFINITY)) b = a, j = i;
}
__device__ __forceinline__ void warp_best(float& b, int& j) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) better(b, j, __shfl_xor_sync(0xffffffffu, b, o), __shfl_xor_sync(0xffffffffu, j, o));
}
// The row's part of a list; nothing, with the status word set, where it lies outside.
__device__ __forceinline__ bool row_range(const int32_t* ptr, uint32_t row, uint32_t n, uint32_t* a, uint32_t* b, uint32_t* status) {
    *a = 0;
    *b = n;
    if (!ptr) return true;
    const int lo = ptr[row], hi = ptr[row + 1];
    if (lo < 0 || hi < lo || (uint32_t)hi > n) {
        *a = *b = 0;
        *(volatile uint32_t*)status = LOGITS_BAD_LIST;
        return false;
    }
    *a = lo;
    *b = hi;
    return true;
}

template <typename T>
__global__ void __launch_bounds__(LG_THREADS) logits_kernel(const LgArgs a) {
    extern __shared__ __align__(16) uint32_t lists[];  // [part] how often, [part] the bias's entry + 1
    __shared__ float best_s[LG_THREADS / 32];
    __shared__ int at_s[LG_THREADS / 32];
    __shared__ struct { float v; int i; } mine;
    pdl_launch_dependents();
    const uint32_t C = lg_size(), cta = lg_rank(), row = blockIdx.x / C, tid = threadIdx.x;
    uint32_t* const times = lists;
    uint32_t* const entry = lists + a.part;
    pdl_wait();
    uint32_t h0 = 0, h1 = 0, b0 = 0, b1 = 0;
    if (a.r.n_history) row_range(a.r.history_ptr, row, a.r.n_history, &h0, &h1, a.status);
    if (a.r.n_bias) row_range(a.r.bias_ptr, row, a.r.n_bias, &b0, &b1, a.status);
    const bool listed = h1 > h0 || b1 > b0;
    const uint32_t* const mask = a.r.mask ? a.r.mask + (size_t)row * a.r.mask_stride : nullptr;
    const T* const x = (const T*)a.x + (size_t)row * a.x_stride;
    T* const out = a.out ? (T*)a.out + (size_t)row * a.out_stride : nullptr;
    float best = -INFINITY;
    int at = 0x7fffffff;
    const uint32_t end = min((cta + 1) * a.slice, a.n);
    for (uint32_t p0 = cta * a.slice; p0 < end; p0 += a.part) {
        const uint32_t m = min(a.part, end - p0);
        if (listed) {
            for (uint32_t i = tid; i < 2 * a.part / 4; i += LG_THREADS) ((uint4*)lists)[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
            for (uint32_t i = h0 + tid; i < h1; i += LG_THREADS) {
                const uint32_t id = (uint32_t)a.r.history[i] - p0;
                if (id < m) atomicAdd(times + id, 1u);
            }
            for (uint32_t i = b0 + tid; i < b1; i += LG_THREADS) {
                const uint32_t id = (uint32_t)a.r.bias_ids[i] - p0;
                if (id < m) atomicMax(entry + id, i - b0 + 1);
            }
            __syncthreads();
        }
        for (uint32_t i = 4 * tid; i < m; i += 4 * LG_THREADS) {
            const uint32_t k = min(4u, m - i), id0 = p0 + i;
            alignas(16) T v[4];
            if (a.aligned && k == 4) {
                if constexpr (sizeof(T) == 4) *(uint4*)v = *(const uint4*)(x + id0);
                else *(uint2*)v = *(const uint2*)(x + id0);
            } else {
                for (uint32_t e = 0; e < k; e++) v[e] = x[id0 + e];
            }
            const uint32_t allowed = mask ? mask[id0 >> 5] >> (id0 & 31) : 0xfu;  // (id0 is a multiple of four)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (e >= (int)k) break;
                float y = as_f32<T>(v[e]);
                if (listed) {
                    const uint32_t c = times[i + e], b = entry[i + e];
                    if (c) {
                        y = y > 0.0f ? __fdiv_rn(y, a.r.repeat) : __fmul_rn(y, a.r.repeat);
                        y = __fsub_rn(y, __fadd_rn(__fmul_rn((float)c, a.r.frequency), a.r.presence));
                    }
                    if (b) y = __fadd_rn(y, a.r.bias[b0 + b - 1]);
                }
                if (!((allowed >> e) & 1)) y = -INFINITY;
                v[e] = rounded<T>(y);
                better(best, at, as_f32<T>(v[e]), (int)(id0 + e));
            }
            if (out) {
                if (a.aligned && k == 4) {
                    if constexpr (sizeof(T) == 4) *(uint4*)(out + id0) = *(const uint4*)v;
                    else *(uint2*)(out + id0) = *(const uint2*)v;
                } else {
                    for (uint32_t e = 0; e < k; e++) out[id0 + e] = v[e];
                }
            }
        }
        if (listed) __syncthreads();
    }
    if (!a.pick) return;
    warp_best(best, at);
    if ((tid & 31) == 0) {
        best_s[tid >> 5] = best;
        at_s[tid >> 5] = at;
    }
    __syncthreads();
    if (tid < 32) {
        best = tid < LG_THREADS / 32 ? best_s[tid] : -INFINITY;
        at = tid < LG_THREADS / 32 ? at_s[tid] : 0x7fffffff;
        warp_best(best, at);
        if (tid == 0) {
            mine.v = best;
            mine.i = at;
        }
    }
    if (C > 1) {
        lg_sync();
        if (cta == 0 && tid < 32) {
            best = tid < C ? __uint_as_float(lg_peer(&mine.v, tid)) : -INFINITY;
            at = tid < C ? (int)lg_peer(&mine.i, tid) : 0x7fffffff;
            warp_best(best, at);
        }
        lg_sync();  // (nobody ends before it has been read)
    }
    if (cta == 0 && tid == 0) a.pick[row] = at == 0x7fffffff ? -1 : at;
}

template <typename T>
cudaError_t logits_t(LgArgs& a, uint32_t t, cudaStream_t st, bool pdl) {
    const uint32_t C = std::min<uint32_t>(16, (a.n + LG_PART - 1) / LG_PART);
    if (t > 0x7fffffffu / C) return cudaErrorInvalidValue;
    a.slice = ((a.n + C - 1) / C + 31) & ~31u;
    const uint32_t parts = (a.slice + LG_PART - 1) / LG_PART;
    a.part = ((a.slice + parts - 1) / parts + 31) & ~31u;
    const size_t smem = a.r.n_history || a.r.n_bias ? (size_t)a.part * 8 : 0;
    auto kern = logits_kernel<T>;
    if (cudaError_t e = ensure_dynamic_smem((const void*)kern, smem, 0); e != cudaSuccess) return e;
    if (cudaError_t e = cudaFuncSetAttribute((const void*)kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); e != cudaSuccess) return e;
    const size_t unit = 4 * sizeof(T);
    a.aligned = (((uintptr_t)a.x | (uintptr_t)a.out | a.x_stride * sizeof(T) | (a.out ? a.out_stride * sizeof(T) : 0)) & (unit - 1)) == 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(t * C);
    cfg.blockDim = dim3(LG_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

__global__ void advance_kernel(const int32_t* pick, int* token, int* out_tokens, int32_t* history, int32_t* history_ptr, uint32_t* sp) {
    pdl_launch_dependents();
    pdl_wait();
    const int id = max(*pick, 0);
    *token = id;
    out_tokens[sp[2]] = id;
    history[history_ptr[1]] = id;
    history_ptr[1] += 1;
    sp[2] += 1;
    sp[0] += 1;
}

}  // namespace

cudaError_t launch_advance(const int32_t* pick, int* token, int* out_tokens, int32_t* history, int32_t* history_ptr, uint32_t* sp, cudaStream_t st, bool pdl) {
    return launch_k(advance_kernel, dim3(1), dim3(1), 0, st, pdl, pick, token, out_tokens, history, history_ptr, sp);
}

cudaError_t launch_logits(const void* x, void* out, int dtype, size_t x_stride, size_t out_stride, uint32_t t, uint32_t n, const LogitRulesDev& r, int32_t* pick,
                          uint32_t* status, cudaStream_t st, bool pdl) {
    if (t == 0 || n == 0) return cudaSuccess;
    if (n > 0x7ffffff0u) return cudaErrorInvalidValue;
    LgArgs a{};
    a.x = x;
    a.out = out;
    a.x_stride = x_stride;
    a.out_stride = out_stride;
    a.n = n;
    a.r = r;
    if (r.repeat == 1.0f && r.frequency == 0.0f && r.presence == 0.0f) a.r.n_history = 0;  // (nothing to change)
    a.pick = pick;
    a.status = status;
    switch (dtype) {
        case B2_F32: return logits_t<float>(a, t, st, pdl);
        case B2_BF16: return logits_t<__nv_bfloat16>(a, t, st, pdl);
        case B2_F16: return logits_t<__half>(a, t, st, pdl);
    }
    return cudaErrorInvalidValue;
}

}  // namespace b2
