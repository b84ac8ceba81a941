// Rows of logits before a token is chosen (the reference does this on the host, src/sampler.rs): for every token that the row's history has c > 0 times
//   l = l > 0 ? l / repeat : l * repeat,  l -= frequency c + presence,
// then a bias where the row's list has one (the last entry of a token counts), -inf where the mask does not allow it; and the first largest.
// Every operation is a rounding of f32 of its own, so the values are those of the same formulas anywhere; 16-bit rows are rounded once at the end, and
// the choice is among what is stored.
//
// A cluster of CTAs has a row, a slice of the tokens each. What the lists say of a slice's tokens is counted in shared memory (integers, so the order of the
// atomics does not matter), every list read once by each CTA; the tokens that are on one are listed by whoever counts them first and changed, and the pass over the
// logits, which were asked for before all that, takes those values where there are any. The CTAs' largest values go to the first one's shared memory.
// What bounds it: a CTA's chain for a part (a list's bounds, its tokens, the counts, the changes, the pass), some 6 us for two to four CTAs an SM at a time, and
// whole waves of them. Replays (cold caches 9.0, 24.6 and 28.3 us): one row of 128256 with 1500 tokens of history 6.9 us, 64 rows with 700 15.5 us (4.3 TB/s of 66.8 MB, half of it from L2), 256 bf16 rows of 32064
// under all rules 22.6 us. Steps: changes made in the pass itself, where every warp met one, 8.3 / 32.7 / 39.1; tokens listed one warp's vote at a time 7.3 / 21.5 / 34
// (gathered ahead of their counting, too, 8.1 / 25 / 39.5: the barriers cost more); not a CTA for every part of a row but whole waves of them 6.8 / 15.7 / 28.4; a warp's
// votes for all of a thread's tokens at once 6.9 / 15.4 / 23.3; 16-bit logits two at a time 7.0 / 15.5 / 22.6.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "async_copy.cuh"
#include "kernels.h"
#include "pdl.cuh"

namespace b2 {

using namespace acopy;

namespace {

constexpr int LG_PART = 8192;  // tokens that are counted at a time

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
template <typename T>
using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
template <typename T>
__device__ __forceinline__ uint32_t bits_of(float v) {
    const T t = rounded<T>(v);
    return *(const unsigned short*)&t;
}
// What a token of a list has become, never zero: the complement of its bits in f32 (NaN as the one whose complement is not zero), or the bits of its rounding and one more.
template <typename T>
__device__ __forceinline__ uint32_t mark(float y) {
    if constexpr (sizeof(T) == 2) return bits_of<T>(y) | 0x10000u;
    else return ~__float_as_uint(y == y ? y : NAN);
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
// Into another CTA's shared memory, counted on its barrier.
__device__ __forceinline__ void lg_push(void* p, uint32_t v, uint64_t* bar, uint32_t cta) {
    uint32_t a, m;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(cta));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(m) : "r"(smem_addr(bar)), "r"(cta));
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.u32 [%0], %1, [%2];" ::"r"(a), "r"(v), "r"(m) : "memory");
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

// Up to 16 bytes of a row.
template <typename T>
__device__ __forceinline__ uint4 load_group(const T* p, uint32_t k, bool aligned) {
    constexpr uint32_t V = 16 / sizeof(T);
    if (aligned && k == V) return *(const uint4*)p;
    alignas(16) T v[V];
#pragma unroll
    for (uint32_t e = 0; e < V; e++) v[e] = e < k ? p[e] : rounded<T>(-INFINITY);
    return *(const uint4*)v;
}
template <typename T>
__device__ __forceinline__ void store_group(T* p, uint4 w, uint32_t k, bool aligned) {
    constexpr uint32_t V = 16 / sizeof(T);
    if (aligned && k == V) {
        *(uint4*)p = w;
        return;
    }
    alignas(16) T v[V];
    *(uint4*)v = w;
#pragma unroll
    for (uint32_t e = 0; e < V; e++)
        if (e < k) p[e] = v[e];
}

// The slice's logits are asked for before the lists are counted: a thread has 16 tokens of a part, by 16 bytes.
template <typename T, int LG_THREADS, bool TIMES, bool ENTRY>
__global__ void __launch_bounds__(LG_THREADS, 1024 / LG_THREADS) logits_kernel(const LgArgs a) {
    constexpr uint32_t V = 16 / sizeof(T), GROUPS = LG_PART / (LG_THREADS * V);
    // [part] how often (TIMES), [part] the bias's entry + 1 (ENTRY), and the tokens that are on a list, each once, u16. What the rules make of such a token then
    // takes the place of its count (or entry), see mark().
    extern __shared__ __align__(16) uint32_t lists[];
    __shared__ uint32_t n_listed;
    __shared__ float best_s[LG_THREADS / 32];
    __shared__ int at_s[LG_THREADS / 32];
    __shared__ uint32_t theirs[2][16];  // the first CTA's: the others' largest values and their tokens
    __shared__ uint64_t come;
    pdl_launch_dependents();
    const uint32_t C = lg_size(), cta = lg_rank(), row = blockIdx.x / C, tid = threadIdx.x;
    if (C > 1) {
        if (cta == 0 && tid == 0) {
            bar_init(&come, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            bar_expect_tx(&come, (C - 1) * 8);
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (waited for ahead of the stores below)
    }
    uint32_t* const times = lists;
    uint32_t* const entry = lists + (TIMES ? a.part : 0);
    uint16_t* const listed = (uint16_t*)(lists + (TIMES + ENTRY) * a.part);
    pdl_wait();
    uint32_t h0 = 0, h1 = 0, b0 = 0, b1 = 0;
    if (TIMES) row_range(a.r.history_ptr, row, a.r.n_history, &h0, &h1, a.status);
    if (ENTRY) row_range(a.r.bias_ptr, row, a.r.n_bias, &b0, &b1, a.status);
    const uint32_t* const mask = a.r.mask ? a.r.mask + (size_t)row * a.r.mask_stride : nullptr;
    const T* const x = (const T*)a.x + (size_t)row * a.x_stride;
    T* const out = a.out ? (T*)a.out + (size_t)row * a.out_stride : nullptr;
    float best = -INFINITY;
    int at = 0x7fffffff;
    const uint32_t end = min((cta + 1) * a.slice, a.n);
    // a thread's tokens of the two lists, for every part; what is behind them goes through `listed`
    constexpr int AHEAD = TIMES ? (LG_THREADS == 512 ? 8 : 4) : 0, BIASES = ENTRY ? 1 : 0;
    uint32_t ids[AHEAD + BIASES + 1];
    for (uint32_t p0 = cta * a.slice; p0 < end; p0 += a.part) {
        const uint32_t m = min(a.part, end - p0);
        if (p0 == cta * a.slice) {
#pragma unroll
            for (int i = 0; i < AHEAD + BIASES; i++) {
                const uint32_t j = i < AHEAD ? h0 + tid + i * LG_THREADS : b0 + tid + (i - AHEAD) * LG_THREADS;
                ids[i] = i < AHEAD ? (j < h1 ? (uint32_t)a.r.history[j] : 0xffffffffu) : j < b1 ? (uint32_t)a.r.bias_ids[j] : 0xffffffffu;
            }
        }
        uint4 w[GROUPS];
        uint32_t allowed[GROUPS];
#pragma unroll
        for (uint32_t gi = 0; gi < GROUPS; gi++) {
            const uint32_t i = (gi * LG_THREADS + tid) * V;
            w[gi] = i < m ? load_group(x + p0 + i, min(V, m - i), a.aligned) : make_uint4(0, 0, 0, 0);
            allowed[gi] = mask && i < m ? mask[(p0 + i) >> 5] >> ((p0 + i) & 31) : 0xffu;  // (p0 + i is a multiple of V)
        }
        if (TIMES || ENTRY) {
            for (uint32_t i = tid; i < (TIMES + ENTRY) * a.part / 4; i += LG_THREADS) ((uint4*)lists)[i] = make_uint4(0, 0, 0, 0);
            if (tid == 0) n_listed = 0;
            __syncthreads();
            const uint32_t lane = tid & 31;
            auto put = [&](bool first, uint32_t id) {  // (the whole warp)
                const uint32_t all = __ballot_sync(0xffffffffu, first);
                if (all == 0) return;
                uint32_t at0 = 0;
                if (lane == 0) at0 = atomicAdd(&n_listed, (uint32_t)__popc(all));
                at0 = __shfl_sync(0xffffffffu, at0, 0);
                if (first) listed[at0 + __popc(all & ((1u << lane) - 1))] = (uint16_t)id;
            };
            if (TIMES) {
                uint32_t all[AHEAD + 1], mine = 0;  // the first that finds a token puts it on the list
#pragma unroll
                for (int i = 0; i < AHEAD; i++) {
                    const uint32_t id = ids[i] != 0xffffffffu && ids[i] - p0 < m ? ids[i] - p0 : m;
                    all[i] = __ballot_sync(0xffffffffu, id < m && atomicAdd(times + id, 1u) == 0);
                    mine += __popc(all[i]);
                }
                uint32_t at0 = 0;
                if (lane == 0 && mine) at0 = atomicAdd(&n_listed, mine);
                at0 = __shfl_sync(0xffffffffu, at0, 0);
#pragma unroll
                for (int i = 0; i < AHEAD; i++) {
                    if ((all[i] >> lane) & 1) listed[at0 + __popc(all[i] & ((1u << lane) - 1))] = (uint16_t)(ids[i] - p0);
                    at0 += __popc(all[i]);
                }
                for (uint32_t i = h0 + tid - lane + AHEAD * LG_THREADS; i < h1; i += LG_THREADS) {
                    const uint32_t id = i + lane < h1 ? (uint32_t)a.r.history[i + lane] - p0 : m;
                    put(id < m && atomicAdd(times + id, 1u) == 0, id);
                }
            }
            if (ENTRY) {
                if (TIMES) __syncthreads();
                for (uint32_t i = b0 + tid - lane; i < b1; i += LG_THREADS) {
                    const uint32_t given = i == b0 + tid - lane ? ids[AHEAD] : i + lane < b1 ? (uint32_t)a.r.bias_ids[i + lane] : 0xffffffffu;
                    const uint32_t id = given != 0xffffffffu && given - p0 < m ? given - p0 : m;
                    put(id < m && atomicMax(entry + id, i + lane - b0 + 1) == 0 && !(TIMES && times[id]), id);
                }
            }
            __syncthreads();
            auto change = [&](uint32_t id, float y) {
                const uint32_t c = TIMES ? times[id] : 0, b = ENTRY ? entry[id] : 0;
                if (c) {
                    y = y > 0.0f ? __fdiv_rn(y, a.r.repeat) : __fmul_rn(y, a.r.repeat);
                    y = __fsub_rn(y, __fadd_rn(__fmul_rn((float)c, a.r.frequency), a.r.presence));
                }
                if (b) y = __fadd_rn(y, a.r.bias[b0 + b - 1]);
                lists[id] = mark<T>(y);
            };
            for (uint32_t j = tid; j < n_listed; j += LG_THREADS) change(listed[j], as_f32<T>(x[p0 + listed[j]]));
            __syncthreads();
        }
#pragma unroll
        for (uint32_t gi = 0; gi < GROUPS; gi++) {
            const uint32_t i = (gi * LG_THREADS + tid) * V, k = i < m ? min(V, m - i) : 0u;
            if (k == 0) continue;
            alignas(16) T v[V];
            float top;
            if constexpr (sizeof(T) == 2) {  // two at a time
                uint32_t x[4] = {w[gi].x, w[gi].y, w[gi].z, w[gi].w};
                const uint32_t none = bits_of<T>(-INFINITY);
                T2<T> high;
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) {
                    uint32_t lo = x[e], hi = x[e] >> 16;
                    if (TIMES || ENTRY) {
                        const uint2 f = *(const uint2*)(lists + i + 2 * e);
                        lo = f.x ? f.x : lo;
                        hi = f.y ? f.y : hi;
                    }
                    if (!((allowed[gi] >> (2 * e)) & 1)) lo = none;
                    if (!((allowed[gi] >> (2 * e + 1)) & 1)) hi = none;
                    x[e] = __byte_perm(lo, hi, 0x5410);
                    high = e ? __hmax2(high, *(const T2<T>*)&x[e]) : *(const T2<T>*)&x[e];  // (what lies behind the row is -inf; NaN is passed over)
                }
                top = fmaxf(as_f32<T>(high.x), as_f32<T>(high.y));
                *(uint4*)v = make_uint4(x[0], x[1], x[2], x[3]);
            } else {
                *(uint4*)v = w[gi];
                if (TIMES || ENTRY) {
                    const uint4 f = *(const uint4*)(lists + i);
                    if (f.x) v[0] = __uint_as_float(~f.x);
                    if (f.y) v[1] = __uint_as_float(~f.y);
                    if (f.z) v[2] = __uint_as_float(~f.z);
                    if (f.w) v[3] = __uint_as_float(~f.w);
                }
                top = -INFINITY;
#pragma unroll
                for (uint32_t e = 0; e < V; e++) {
                    if (!((allowed[gi] >> e) & 1)) v[e] = -INFINITY;
                    top = fmaxf(top, v[e]);
                }
            }
            if (top > best) {  // (seldom, and the first of equals)
                best = top;
#pragma unroll
                for (int e = (int)V - 1; e >= 0; e--)
                    if (as_f32<T>(v[e]) == top) at = (int)(p0 + i) + e;
            }
            if (out) store_group(out + p0 + i, *(const uint4*)v, k, a.aligned);
        }
        if ((TIMES || ENTRY) && p0 + a.part < end) __syncthreads();
    }
    if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (!a.pick) return;
    warp_best(best, at);
    if ((tid & 31) == 0) {
        best_s[tid >> 5] = best;
        at_s[tid >> 5] = at;
    }
    __syncthreads();
    if (tid >= 32) return;
    best = tid < LG_THREADS / 32 ? best_s[tid] : -INFINITY;
    at = tid < LG_THREADS / 32 ? at_s[tid] : 0x7fffffff;
    warp_best(best, at);
    if (cta > 0) {
        if (tid == 0) {
            lg_push(&theirs[0][cta], __float_as_uint(best), &come, 0);
            lg_push(&theirs[1][cta], (uint32_t)at, &come, 0);
        }
        return;
    }
    if (C > 1) {
        if (!bar_wait<true>(&come, 0)) *(volatile uint32_t*)a.status = KV8_TIMEOUT;
        if (tid > 0) {
            best = tid < C ? __uint_as_float(theirs[0][tid]) : -INFINITY;
            at = tid < C ? (int)theirs[1][tid] : 0x7fffffff;
        }
        warp_best(best, at);
    }
    if (cta == 0 && tid == 0) a.pick[row] = at == 0x7fffffff ? -1 : at;
}

// CTAs of a row, as many as end it first: waves of CTAs times their parts, and 0.4 of a part for a CTA's start and end. us, this / as many CTAs as a row has parts: 64 rows
// of 128256 with 700 tokens of history 21.8 / 31.2 (from memory), 256 bf16 rows of 32064 with 4000 and 300 biases 28.4 / 33.5, 1000 with 500 56 / 67.
double lg_split(uint32_t t, uint32_t n, uint32_t lists, uint32_t threads, uint32_t* C) {
    const uint32_t parts = (n + LG_PART - 1) / LG_PART;
    const uint32_t fit = 148 * std::min<uint32_t>(1024 / threads, lists ? 227 * 1024 / (LG_PART * (4 * lists + 2) + 2048) : 4);
    double least = 0.0;
    for (uint32_t c = 1; c <= std::min<uint32_t>(16, parts); c = c == 8 ? 16 : c + 1) {
        const uint32_t at_once = c == 16 ? fit * 3 / 4 : fit;  // (fourteen clusters of sixteen fit the chip, and hardly more of nine to fifteen)
        const double cost = (double)(((size_t)t * c + at_once - 1) / at_once) * ((parts + c - 1) / c + 0.4);
        if (c == 1 || cost < least) {
            *C = c;
            least = cost;
        }
    }
    return least;
}

template <typename T, int LG_THREADS>
cudaError_t logits_n(LgArgs& a, uint32_t t, uint32_t C, cudaStream_t st, bool pdl) {
    if (t > 0x7fffffffu / C) return cudaErrorInvalidValue;
    a.slice = ((a.n + C - 1) / C + 31) & ~31u;
    const uint32_t parts = (a.slice + LG_PART - 1) / LG_PART;
    a.part = ((a.slice + parts - 1) / parts + 31) & ~31u;
    const size_t smem = a.r.n_history || a.r.n_bias ? (size_t)a.part * (4 * ((a.r.n_history != 0) + (a.r.n_bias != 0)) + 2) : 0;
    auto kern = a.r.n_history ? (a.r.n_bias ? logits_kernel<T, LG_THREADS, true, true> : logits_kernel<T, LG_THREADS, true, false>)
                              : (a.r.n_bias ? logits_kernel<T, LG_THREADS, false, true> : logits_kernel<T, LG_THREADS, false, false>);
    if (cudaError_t e = ensure_dynamic_smem((const void*)kern, smem, 0); e != cudaSuccess) return e;
    if (cudaError_t e = cudaFuncSetAttribute((const void*)kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); e != cudaSuccess) return e;
    a.aligned = (((uintptr_t)a.x | (uintptr_t)a.out | a.x_stride * sizeof(T) | (a.out ? a.out_stride * sizeof(T) : 0)) & 15) == 0;
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

template <typename T>
cudaError_t logits_t(LgArgs& a, uint32_t t, cudaStream_t st, bool pdl) {
    // CTAs of 512 threads, two an SM, or of 256, four an SM (two where shared memory has to hold two lists), which take 1.35 times as long for a part and, with four tokens a thread
    // at a time, are for short lists. 512 / 256 threads, us: one row of 128256 7.0 / 9.2, 16 rows with 700 tokens of history 11.3 / 8.9, 32 11.6 / 14.0, 64 24.4 / 21.6,
    // with 4000 30.6 / 34.5; 1000 bf16 rows of 32064 with 500 79 / 56.
    const uint32_t lists = (a.r.n_history != 0) + (a.r.n_bias != 0);
    uint32_t C = 1, C_small = 1;
    const bool small = lg_split(t, a.n, lists, 512, &C) > 1.35 * lg_split(t, a.n, lists, 256, &C_small) && ((size_t)a.r.n_history + a.r.n_bias) / t < 1024;
    return small ? logits_n<T, 256>(a, t, C_small, st, pdl) : logits_n<T, 512>(a, t, C, st, pdl);
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
