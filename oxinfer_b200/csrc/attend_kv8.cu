// Attention over the 8-bit cache (kv8.cuh): y = sum_j p_j v_j with p = softmax over the keys that a query sees of
//   cap tanh(scale q.k / cap) + slope (j - position)      (cap 0: no cap; no slopes: no bias)
// for the queries of several sequences, one token each or many. Key j is seen by the query at position p where j <= p or j < prefix, and, with a window,
// p - j < window.
//
// A tile of rows (query heads of a KV head, token by token) is taken by a cluster of CTAs over all of its keys; every warp of them takes blocks of 32 keys
// in turn, each with a ring of units of its own (one bulk copy a unit: header, keys and values lie side by side), a running maximum and sums, and the
// partial sums are added warp by warp in shared memory and CTA by CTA over the cluster, in a fixed order.
//
// The products are mma.sync.m16n8k16 on the integers as f16, which is exact; a unit's scales multiply the scores and the sums of a unit in f32. With eight rows a
// tile the instruction's other eight carry the second f16 term of the queries (each row first multiplied by a power of two) and of the probabilities, 22 bits of
// both: results of f32 accuracy at no further cost. Tiles of sixteen rows (f16 and bf16 results of many rows) have one term.
//
// What bounds it (times of replays; with cold caches one token over 2048 keys takes 10.3, over 131071 59, the 64 sequences with a cap 73): long contexts HBM, at 4.3 to 4.9 TB/s of a measured 6.5 (750 instructions a block of 128 dimensions keep half of the issue slots busy, with three warps a scheduler to
// cover the softmax's chain); short ones latency: a launch, the first block, two to four blocks a warp one behind the other, the cluster's sums. 32 heads of 8 KV heads of 128, us: one
// token over 2048 keys 7.9, over 131071 54.9; 64 sequences of up to 4096 with a cap 67.1. f32 rows of a prompt take eight-row tiles, too: 2048 tokens behind 2048 820, 16-bit rows (attend_kv8_rows.cu) 112. Steps: two CTAs an SM 110, three 84 (131071: 121), blocks dealt out over all of the GPU 76 and
// 68 (55), caps and sums two values an instruction 68.5 instead of 78.7 with a cap.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "async_copy.cuh"
#include "kv8.cuh"
#include "pdl.cuh"

namespace b2 {

using namespace acopy;
using namespace kv8;

namespace {

constexpr int AK_WARPS = 4, AK_THREADS = AK_WARPS * 32;
constexpr uint32_t DEALT_CTAS = 3 * 148, DEALT_LEAST = 4;  // three an SM; blocks of a warp
template <int HD>
constexpr size_t DEALT_FLOAT4 = 8 * HD / 4 + 8;  // of a place: the sums of eight rows, their largest scores and denominators
constexpr float P_BITS = 14.0f;  // probabilities are held 2^14 times as large: what is below 2^-28 of a row's largest loses bits, not before
// Sums of probabilities times values are held 2^40 times as small, so that they stay finite where the values are (P_BITS, and up to 2^26 keys of a row); a scale is at least 2^-100.
constexpr float SUM_DOWN = 0x1p-40f, SUM_UP = 0x1p40f;

template <int HD, int TERMS>
struct AkShared {
    static constexpr uint32_t UNIT = unit_bytes(HD);
    static constexpr int CTAS = TERMS == 2 ? 3 : 2;                // of an SM (registers)
    static constexpr int STAGES = (TERMS == 2 ? 2 : 3) * (HD == 128 ? 1 : 2);
    static constexpr uint32_t RING = STAGES * UNIT;
    static constexpr uint32_t ML = AK_WARPS * RING;                // [16] largest, [16] denominators of the CTA, then of the warps [warp][16][2]
    static constexpr uint32_t BARS = ML + (2 + 2 * AK_WARPS) * 16 * 4;
    static constexpr uint32_t BYTES = BARS + AK_WARPS * STAGES * 8;
    static_assert(RING >= 16 * HD * 4, "a warp's sums take its ring's place");
    static_assert(CTAS * (BYTES + 1024) <= 228 * 1024);
};

struct AkArgs {
    Kv8Cache c;
    Kv8Seqs sq;
    const void* q;
    void* out;
    size_t q_stride, out_stride;
    uint32_t G, tiles, window;
    float c2, cap2, cap_in;  // scale in powers of two; cap in powers of two, and 2 / cap of scores in powers of two
    const float* slopes;
    const int32_t* prefix;
    int aligned;
    float4* work;  // dealt-out launches: sums of units of work that several CTAs share
    uint32_t* status;
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same from zero (no registers to clear first).
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// Bytes q + 128 as f16: 1024 + byte by its bits, then minus 1152 (exact).
__device__ __forceinline__ uint32_t two_halves(uint32_t w, uint32_t sel) {
    const uint32_t x = __byte_perm(w, 0x64646464u, sel);
    const __half2 h = __hsub2(*(const __half2*)&x, __half2half2(__ushort_as_half(0x6480)));
    return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t low_half(uint32_t w) { return two_halves(w, 0x4140u); }
__device__ __forceinline__ uint32_t high_half(uint32_t w) { return two_halves(w, 0x4342u); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
}
// What f16 leaves of two values.
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
    const float2 f = __half22float2(*(const __half2*)&hi), rest = add2(make_float2(a, b), make_float2(-f.x, -f.y));
    return pack(rest.x, rest.y);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// cap tanh(y / cap), y and the result in powers of two, of eight: up to |z| = 1 by an odd polynomial fitted at Chebyshev nodes of z^2 (off by 1.5e-7), beyond by an exponential.
__device__ __forceinline__ void capped(float2 (&y)[4], float cap2, float cap_in) {
    float2 z[4], x[4];
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        z[j] = mul2(y[j], both(0.5f * 0.69314718f * cap_in));
        most = max3(most, fabsf(z[j].x), fabsf(z[j].y));
        const float2 z2 = mul2(z[j], z[j]);
        float2 p = fma2(z2, both(1.04555360e-3f), both(-6.21706992e-3f));
        p = fma2(z2, p, both(2.03055199e-2f));
        p = fma2(z2, p, both(-5.34651764e-2f));
        p = fma2(z2, p, both(1.33253977e-1f));
        p = fma2(z2, p, both(-3.33328575e-1f));
        x[j] = mul2(y[j], fma2(z2, p, both(9.9999994e-1f)));
    }
    if (most > 1.0f) {
        auto far = [&](float y) { return cap2 * (1.0f - __fdividef(2.0f, 1.0f + ex2(y * cap_in))); };
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (fabsf(z[j].x) > 1.0f) x[j].x = far(y[j].x);
            if (fabsf(z[j].y) > 1.0f) x[j].y = far(y[j].y);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) y[j] = x[j];
}
template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v, bool aligned) {
    alignas(16) T t[4];
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) t[i] = f[i];
        else if constexpr (std::is_same<T, __half>::value) t[i] = __float2half_rn(f[i]);
        else t[i] = __float2bfloat16_rn(f[i]);
    }
    if (aligned) {
        if constexpr (sizeof(T) == 4) *(float4*)p = v;
        else *(uint2*)p = *(const uint2*)t;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = t[i];
    }
}
__device__ __forceinline__ uint32_t peer(const void* p, uint32_t cta) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(cta));
    return r;
}
__device__ __forceinline__ float4 peer_f4(const void* p, uint32_t cta) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer(p, cta)) : "memory");
    return v;
}
__device__ __forceinline__ float2 peer_f2(const void* p, uint32_t cta) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(peer(p, cta)) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float weight_of(float m, float most) { return ex2(m - (most == -INFINITY ? 0.0f : most)); }

// Dealt-out launches. The blocks of all units (tile of rows, KV head) of all sequences lie one behind another, and CTA i of n takes i W / n .. (i + 1) W / n
// of them; a unit that several CTAs share leaves their sums in memory, two places a CTA (the unit it begins in the middle of, the one it ends in), and
// a kernel behind this one adds them in order. Tiles of a sequence count the same blocks, those that any of its rows sees.
struct Dealt {
    uint32_t lo, blocks, tiles;  // a sequence's first block, blocks of a unit, tiles
};
template <int R>
__device__ __forceinline__ Dealt dealt_of(const AkArgs& a, uint32_t s) {
    Seq q;
    if (s >= a.sq.n_seqs || !sequence(a.sq, s, &q, a.status) || q.count == 0) return Dealt{0, 0, 0};
    const uint32_t lo = a.window && q.start + 1 > a.window ? (q.start + 1 - a.window) / KV8_BLOCK : 0;
    return Dealt{lo, (q.start + q.count + KV8_BLOCK - 1) / KV8_BLOCK - lo, (q.count * a.G + R - 1) / R};
}
__device__ __forceinline__ unsigned long long dealt_weight(const AkArgs& a, const Dealt& d) { return (unsigned long long)d.tiles * a.c.nkv * d.blocks; }
// The weights of all sequences ahead of s, and of all: every thread of the CTA calls this. red: two words a warp.
template <int R>
__device__ __forceinline__ void dealt_sums(const AkArgs& a, uint32_t s, unsigned long long* ahead, unsigned long long* all, unsigned long long* red) {
    unsigned long long before = 0, sum = 0;
    for (uint32_t x = threadIdx.x; x < a.sq.n_seqs; x += blockDim.x) {
        const unsigned long long w = dealt_weight(a, dealt_of<R>(a, x));
        sum += w;
        if (x < s) before += w;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if ((threadIdx.x & 31) == 0) {
        red[2 * (threadIdx.x >> 5)] = before;
        red[2 * (threadIdx.x >> 5) + 1] = sum;
    }
    __syncthreads();
    *ahead = *all = 0;
    for (uint32_t i = 0; i < blockDim.x / 32; i++) {
        *ahead += red[2 * i];
        *all += red[2 * i + 1];
    }
    __syncthreads();
}
// The sequence that block `at` of all belongs to, and the weights ahead of it (one warp).
template <int R>
__device__ __forceinline__ uint32_t dealt_find(const AkArgs& a, unsigned long long at, unsigned long long* ahead) {
    unsigned long long before = 0;
    for (uint32_t s0 = 0; s0 < a.sq.n_seqs; s0 += 32) {
        const unsigned long long w = dealt_weight(a, dealt_of<R>(a, s0 + (threadIdx.x & 31)));
        unsigned long long upto = w;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const unsigned long long x = __shfl_up_sync(0xffffffffu, upto, o);
            if ((int)(threadIdx.x & 31) >= o) upto += x;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, before + upto > at);
        if (hit) {
            const int i = __ffs(hit) - 1;
            *ahead = before + __shfl_sync(0xffffffffu, upto - w, i);
            return s0 + i;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    *ahead = before;
    return a.sq.n_seqs;
}
// CTAs that get work: a warp has some blocks, at least
__device__ __forceinline__ uint32_t dealt_ctas(unsigned long long all, uint32_t ctas) { return (uint32_t)min((unsigned long long)ctas, max(all / (DEALT_LEAST * AK_WARPS), 1ull)); }

// A CTA's grid index: (unit of work, CTA of the cluster); a unit: (sequence, tile of rows from the last on, KV head). SPECIAL: a cap or a bias. DEALT: see above.
template <int HD, int TERMS, typename T, bool SPECIAL, bool DEALT>
__global__ void __launch_bounds__(AK_THREADS, TERMS == 2 ? 3 : 2) attend_kv8_kernel(const AkArgs a) {
    using L = AkShared<HD, TERMS>;
    constexpr int R = TERMS == 2 ? 8 : 16, RG = TERMS == 2 ? 1 : 2;  // rows of a tile; a lane's rows
    constexpr int KS = HD / 16, NT = HD / 8, QD = HD / 4, S = L::STAGES;
    extern __shared__ __align__(128) uint8_t smem[];
    pdl_launch_dependents();
    const uint32_t C = DEALT ? 1 : cluster_size(), cta = DEALT ? 0 : cluster_rank();
    const uint32_t work = blockIdx.x / C, rest = work / a.c.nkv, first_tile = a.tiles - 1 - rest % a.tiles;
    uint32_t head = work % a.c.nkv, s = rest / a.tiles;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint8_t* const ring = smem + warp * L::RING;
    uint64_t* const bars = (uint64_t*)(smem + L::BARS) + warp * S;
    float* const sum_s = (float*)smem;  // the CTA's sums, where the first warp's were
    float2* const ml_s = (float2*)(smem + L::ML);  // the CTA's largest scores and denominators
    float* const wm = (float*)(ml_s + 16);         // [warp][16]
    float* const wl = wm + AK_WARPS * 16;
    if (lane == 0) {
        for (int i = 0; i < S; i++) bar_init(&bars[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    pdl_wait();
    Seq seq;
    uint32_t rows = 0, len = 0, prefix = 0;
    auto take = [&](uint32_t x) {  // sequence x
        if (!sequence(a.sq, x, &seq, a.status)) return false;
        rows = seq.count * a.G;
        len = seq.start + seq.count;
        prefix = a.prefix ? (uint32_t)min(max(a.prefix[x], 0), (int)len) : 0;
        return true;
    };
    unsigned long long at = 0, upto = 0, ahead = 0;  // DEALT: the blocks of this CTA, and the weights ahead of the sequence
    Dealt d{};
    if constexpr (DEALT) {
        unsigned long long* const red = (unsigned long long*)wm;
        unsigned long long all;
        dealt_sums<R>(a, 0, &ahead, &all, red);
        const uint32_t n = dealt_ctas(all, gridDim.x);
        if (blockIdx.x >= n || all == 0) return;
        at = all * blockIdx.x / n;
        upto = all * (blockIdx.x + 1) / n;
        s = dealt_find<R>(a, at, &ahead);
        d = dealt_of<R>(a, s);
        take(s);
    } else {
        if (!take(s)) return;  // (the same in every CTA of the cluster)
    }
    const uint32_t NW = C * AK_WARPS, gw = cta * AK_WARPS + warp;
    uint32_t slot = 0, phase = 0, tile = first_tile;
    bool ok = true;

    while (true) {
        uint32_t off = 0, part_end = 0;  // DEALT: the blocks of the unit that this CTA takes
        if constexpr (DEALT) {
            if (at >= upto) break;
            while (at >= ahead + dealt_weight(a, d)) {  // on to the next sequence that has rows
                ahead += dealt_weight(a, d);
                d = dealt_of<R>(a, ++s);
                if (d.blocks) take(s);
            }
            const uint32_t unit = (uint32_t)((at - ahead) / d.blocks);
            off = (uint32_t)((at - ahead) % d.blocks);
            part_end = (uint32_t)min((unsigned long long)d.blocks, off + (upto - at));
            tile = unit / a.c.nkv;
            head = unit % a.c.nkv;
        } else {
            if ((size_t)tile * R >= rows) break;
        }
        const uint32_t row0 = tile * R;
        const uint32_t p_first = seq.start + row0 / a.G, p_last = seq.start + min(row0 + R - 1, rows - 1) / a.G;
        const uint32_t k_end = max(p_last + 1, prefix);                                                // keys below are seen by some row
        const uint32_t k_lo = a.window && p_first + 1 > a.window ? p_first + 1 - a.window : 0;         // keys from here on
        const uint32_t in_lo = a.window && p_last + 1 > a.window ? p_last + 1 - a.window : 0;          // keys from here to in_end are seen by every row
        const uint32_t in_end = max(p_first + 1, prefix);
        const uint32_t b_beg = DEALT ? d.lo + off : k_lo / KV8_BLOCK, b_end = DEALT ? d.lo + part_end : (k_end + KV8_BLOCK - 1) / KV8_BLOCK;

        // copies run ahead: block b_beg + gw + i NW is the warp's i-th
        const uint32_t n_mine = ok && b_end - b_beg > gw ? (b_end - b_beg - gw + NW - 1) / NW : 0;
        uint32_t issued = 0, put = slot;
        int ids = -1;
        auto issue = [&] {  // the whole warp
            if ((issued & 31) == 0) {
                const uint32_t i = issued + lane;
                ids = i < n_mine ? block_of(a.c, a.sq, s, b_beg + gw + i * NW, a.status) : 0;
                if (ids < 0) ids = 0;  // (the status word is set: the results do not count)
            }
            const int id = __shfl_sync(0xffffffffu, ids, issued & 31);
            if (lane == 0) {
                bar_expect_tx(&bars[put], L::UNIT);
                bulk_load(ring + put * L::UNIT, a.c.units + ((size_t)id * a.c.nkv + head) * L::UNIT, L::UNIT, &bars[put]);
            }
            put = put + 1 == S ? 0 : put + 1;
            issued++;
        };
        while (issued < n_mine && issued < S) issue();

        // the queries: a lane has dimensions t QD .. of rows g (and g + 8)
        uint32_t qa[KS][4];
        float qf[RG], slope[RG];
        uint32_t pos[RG];
#pragma unroll
        for (int i = 0; i < RG; i++) {
            const uint32_t r = row0 + g + 8 * i, rc = min(r, rows - 1), tok = rc / a.G, h = head * a.G + rc % a.G;
            pos[i] = seq.start + tok;
            slope[i] = SPECIAL && a.slopes ? a.slopes[h] * 1.44269504f : 0.0f;
            const T* const src = (const T*)a.q + (size_t)(seq.r0 + tok) * a.q_stride + (size_t)h * HD + t * QD;
            float v[QD];
            float top = 0.0f;
            bool odd = false;
#pragma unroll
            for (int e = 0; e < QD; e += 4) {
                float x[4];
                load4(x, src + e, a.aligned);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    v[e + k] = x[k];
                    top = fmaxf(top, fabsf(x[k]));
                    odd = odd || !(fabsf(x[k]) <= FLT_MAX);
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // into [2^13, 2^14): products with 127 stay far from the largest f32, and two f16 terms hold 22 bits
            const int ex = min(max((int)(__float_as_uint(top) >> 23), 40), 254) - 127;
            const float f = pow2(13 - ex);
            qf[i] = pow2(ex - 13) * a.c2;
            if (odd) qf[i] = NAN;
            qf[i] += __shfl_xor_sync(0xffffffffu, odd ? NAN : 0.0f, 1);
            qf[i] += __shfl_xor_sync(0xffffffffu, qf[i] != qf[i] ? NAN : 0.0f, 2);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const float x0 = v[4 * ks] * f, x1 = v[4 * ks + 1] * f, x2 = v[4 * ks + 2] * f, x3 = v[4 * ks + 3] * f;
                qa[ks][i] = pack(x0, x1);
                qa[ks][2 + i] = pack(x2, x3);
                if constexpr (TERMS == 2) {
                    qa[ks][1] = pack_rest(x0, x1, qa[ks][0]);
                    qa[ks][3] = pack_rest(x2, x3, qa[ks][2]);
                }
            }
        }

        float o[NT][2 * RG];
        float m[RG], l[RG];
#pragma unroll
        for (int i = 0; i < RG; i++) m[i] = -INFINITY, l[i] = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2 * RG; e++) o[n][e] = 0.0f;

        uint32_t it = 0;
        for (; it < n_mine; it++) {
            const uint32_t key0 = (b_beg + gw + it * NW) * KV8_BLOCK;
            ok = ok && __all_sync(0xffffffffu, bar_wait(&bars[slot], phase));
            if (!ok) break;
            const uint8_t* const unit = ring + slot * L::UNIT;
            const uint4 hd = *(const uint4*)unit;
            const float k_scale = __uint_as_float(hd.x), v_scale = __uint_as_float(hd.z) * SUM_DOWN;
            const uint32_t bad = hd.y | hd.w;
            float sc[RG][8];  // [row][key 2 t + e of tile j]: 2 j + e
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float d0[4], d1[4];
#pragma unroll
                for (int hf = 0; hf < KS / 4; hf++) {
                    const uint4 w = *(const uint4*)(unit + KV8_HEADER + j * (8 * HD) + hf * 512 + lane * 16);
                    if (hf == 0) {
                        mma16816_first(d0, qa[0], low_half(w.x), high_half(w.x));
                        mma16816_first(d1, qa[1], low_half(w.y), high_half(w.y));
                    } else {
                        mma16816(d0, qa[4 * hf], low_half(w.x), high_half(w.x));
                        mma16816(d1, qa[4 * hf + 1], low_half(w.y), high_half(w.y));
                    }
                    mma16816(d0, qa[4 * hf + 2], low_half(w.z), high_half(w.z));
                    mma16816(d1, qa[4 * hf + 3], low_half(w.w), high_half(w.w));
                }
                const float2 low = add2(make_float2(d0[0], d0[1]), make_float2(d1[0], d1[1])), high = add2(make_float2(d0[2], d0[3]), make_float2(d1[2], d1[3]));
                const float2 first = TERMS == 2 ? add2(low, high) : low;
                sc[0][2 * j] = first.x, sc[0][2 * j + 1] = first.y;
                if (TERMS == 1) sc[RG - 1][2 * j] = high.x, sc[RG - 1][2 * j + 1] = high.y;
            }
            const bool whole = key0 >= in_lo && key0 + KV8_BLOCK <= in_end && bad == 0;  // every row sees every key
            uint32_t ph[RG][4], pl[4];  // probabilities of keys 4 t + 2 j .. : tile j's two
            float shrink[RG];
            bool grown = false;
#pragma unroll
            for (int i = 0; i < RG; i++) {
                float2 y[4];  // keys 16 (j / 2) + 4 t + 2 (j % 2) and the next
#pragma unroll
                for (int j = 0; j < 4; j++) y[j] = mul2(make_float2(sc[i][2 * j], sc[i][2 * j + 1]), both(qf[i] * k_scale));
                if (SPECIAL && a.cap2 > 0.0f) capped(y, a.cap2, a.cap_in);
                if (SPECIAL && a.slopes) {
                    const float first = (float)(int)(key0 + 4 * t - pos[i]);
#pragma unroll
                    for (int j = 0; j < 4; j++) y[j] = fma2(both(slope[i]), add2(both(first), make_float2(16 * (j >> 1) + 2 * (j & 1), 16 * (j >> 1) + 2 * (j & 1) + 1)), y[j]);
                }
                float* const s8 = sc[i];
#pragma unroll
                for (int j = 0; j < 4; j++) s8[2 * j] = y[j].x, s8[2 * j + 1] = y[j].y;
                if (!whole) {
#pragma unroll
                    for (int x = 0; x < 8; x++) {
                        const uint32_t key = key0 + 16 * (x >> 2) + 4 * t + (x & 3);
                        const bool see = key < len && (key <= pos[i] || key < prefix) && (a.window == 0 || (int)(pos[i] - key) < (int)a.window);
                        if ((bad >> (key - key0)) & 1) s8[x] = NAN;
                        if (!see) s8[x] = -INFINITY;
                    }
                }
                float mx = fmaxf(s8[0], s8[1]);
#pragma unroll
                for (int x = 2; x < 8; x += 2) mx = max3(mx, s8[x], s8[x + 1]);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.0f : mn;
                shrink[i] = ex2(m[i] - base);
                grown = grown || mn > m[i];
                m[i] = mn;
                float2 add = both(0.0f);
#pragma unroll
                for (int x = 0; x < 8; x += 2) {
                    const float2 e = add2(make_float2(s8[x], s8[x + 1]), both(P_BITS - base));
                    s8[x] = ex2(e.x), s8[x + 1] = ex2(e.y);
                    add = add2(add, make_float2(s8[x], s8[x + 1]));
                }
                l[i] = fmaf(l[i], shrink[i], add.x + add.y);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    ph[i][j] = pack(sc[i][2 * j], sc[i][2 * j + 1]);
                    if constexpr (TERMS == 2) pl[j] = pack_rest(sc[i][2 * j], sc[i][2 * j + 1], ph[i][j]);
                }
            }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < RG; i++) {
                        const float2 x = mul2(make_float2(o[n][2 * i], o[n][2 * i + 1]), both(shrink[i]));
                        o[n][2 * i] = x.x, o[n][2 * i + 1] = x.y;
                    }
            }
            uint32_t pa[2][4];
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                pa[kk][0] = ph[0][2 * kk];
                pa[kk][2] = ph[0][2 * kk + 1];
                if constexpr (TERMS == 2) {
                    pa[kk][1] = pl[2 * kk];
                    pa[kk][3] = pl[2 * kk + 1];
                } else {
                    pa[kk][1] = ph[RG - 1][2 * kk];
                    pa[kk][3] = ph[RG - 1][2 * kk + 1];
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                const uint4 w = *(const uint4*)(unit + KV8_HEADER + KV8_BLOCK * HD + n / 2 * 512 + lane * 16);
                float d0[4], d1[4];
                mma16816_first(d0, pa[0], low_half(w.x), high_half(w.x));
                mma16816_first(d1, pa[0], low_half(w.z), high_half(w.z));
                mma16816(d0, pa[1], low_half(w.y), high_half(w.y));
                mma16816(d1, pa[1], low_half(w.w), high_half(w.w));
                auto add = [&](float* to, float2 d) {
                    const float2 sum = fma2(d, both(v_scale), make_float2(to[0], to[1]));
                    to[0] = sum.x, to[1] = sum.y;
                };
                if constexpr (TERMS == 2) {
                    add(o[n], add2(make_float2(d0[0], d0[1]), make_float2(d0[2], d0[3])));
                    add(o[n + 1], add2(make_float2(d1[0], d1[1]), make_float2(d1[2], d1[3])));
                } else {
                    add(o[n], make_float2(d0[0], d0[1]));
                    add(o[n] + 2 * RG - 2, make_float2(d0[2], d0[3]));
                    add(o[n + 1], make_float2(d1[0], d1[1]));
                    add(o[n + 1] + 2 * RG - 2, make_float2(d1[2], d1[3]));
                }
            }
            __syncwarp();  // the slot has been read by the whole warp
            if (++slot == S) {
                slot = 0;
                phase ^= 1;
            }
            if (issued < n_mine) issue();
        }
        if (it < n_mine) {
            // A copy did not arrive in time: record it, and give those in flight one more bounded wait each, so that nothing lands in shared memory that has
            // been handed on. The warp takes no more keys, and meets the others at every barrier.
            if (lane == 0) *(volatile uint32_t*)a.status = KV8_TIMEOUT;
            for (; it < issued; it++) {
                bar_wait(&bars[slot], phase);
                if (++slot == S) {
                    slot = 0;
                    phase ^= 1;
                }
            }
            __syncwarp();
        }

        // the warp's sums, in its ring (no copy is in flight)
#pragma unroll
        for (int i = 0; i < RG; i++) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if (t == 0) {
                wm[warp * 16 + g + 8 * i] = m[i];
                wl[warp * 16 + g + 8 * i] = l[i];
            }
#pragma unroll
            for (int n = 0; n < NT; n++) *(float2*)((float*)ring + (g + 8 * i) * HD + n * 8 + 2 * t) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
        }
        __syncthreads();
        constexpr int ITEMS = R * HD / 4;
        auto finish = [&](int item, float4 v, float den) {
            const uint32_t r = row0 + item / (HD / 4);
            if (r >= rows) return;
            const float inv = den > 0.0f || den != den ? SUM_UP / den : 0.0f;  // (a row that sees nothing: zeros)
            T* const to = (T*)a.out + (size_t)(seq.r0 + r / a.G) * a.out_stride + (size_t)(head * a.G + r % a.G) * HD + item % (HD / 4) * 4;
            store4<T>(to, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv), a.aligned);
        };
        for (int item = tid; item < ITEMS; item += AK_THREADS) {
            const int r = item / (HD / 4);
            float M = -INFINITY, den = 0.0f;
#pragma unroll
            for (int w = 0; w < AK_WARPS; w++) M = fmaxf(M, wm[w * 16 + r]);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < AK_WARPS; w++) {
                const float k = weight_of(wm[w * 16 + r], M);
                const float4 x = ((const float4*)(smem + w * L::RING))[item];
                v.x = fmaf(k, x.x, v.x), v.y = fmaf(k, x.y, v.y), v.z = fmaf(k, x.z, v.z), v.w = fmaf(k, x.w, v.w);
                den = fmaf(k, wl[w * 16 + r], den);
            }
            if (DEALT && (off > 0 || part_end < d.blocks)) {
                float4* const to = a.work + (size_t)(2 * blockIdx.x + (off > 0 ? 0 : 1)) * DEALT_FLOAT4<HD>;
                to[item] = v;
                if (item % (HD / 4) == 0) to[R * HD / 4 + r] = make_float4(M, den, 0.0f, 0.0f);
            } else if (C == 1) {
                finish(item, v, den);
            } else {
                ((float4*)sum_s)[item] = v;
                if (item % (HD / 4) == 0) ml_s[r] = make_float2(M, den);
            }
        }
        if (C > 1) {
            cluster_sync();
            for (int item = (int)cta * AK_THREADS + tid; item < ITEMS; item += (int)C * AK_THREADS) {
                const int r = item / (HD / 4);
                // (eight CTAs' words in flight at once)
                float M = -INFINITY, den = 0.0f;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                for (uint32_t k0 = 0; k0 < C; k0 += 8) {
                    float2 ml[8];
                    float4 x[8];
#pragma unroll
                    for (uint32_t k = 0; k < 8; k++) {
                        ml[k] = make_float2(-INFINITY, 0.0f);
                        x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (k0 + k < C) {
                            ml[k] = peer_f2(ml_s + r, k0 + k);
                            x[k] = peer_f4((const float4*)sum_s + item, k0 + k);
                        }
                    }
                    float m = M;
#pragma unroll
                    for (int k = 0; k < 8; k++) m = fmaxf(m, ml[k].x);
                    const float keep = weight_of(M, m);
                    v = make_float4(v.x * keep, v.y * keep, v.z * keep, v.w * keep);
                    den *= keep;
                    M = m;
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const float w = weight_of(ml[k].x, M);
                        v.x = fmaf(w, x[k].x, v.x), v.y = fmaf(w, x[k].y, v.y), v.z = fmaf(w, x[k].z, v.z), v.w = fmaf(w, x[k].w, v.w);
                        den = fmaf(w, ml[k].y, den);
                    }
                }
                finish(item, v, den);
            }
            cluster_sync();  // nobody ends, or writes its sums anew, before its peers have read them
        } else {
            __syncthreads();
        }
        // the rings are free again: their copies are asynchronous writes behind these reads and writes
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        if constexpr (DEALT) at += part_end - off;
        else tile += a.tiles;
    }
}

// Adds the sums of the units that several CTAs shared, `ctas` of them ahead of it. A thread has four outputs. Grid: (sequence, tile, KV head) and, ROW (few units,
// shared by many CTAs), row of the tile: eight groups of threads take a place in turn then, and their sums are added in order.
template <int HD, bool ROW, typename T>
__global__ void __launch_bounds__(2 * HD) attend_kv8_join(const AkArgs a, uint32_t ctas) {
    constexpr int R = 8, ITEMS = R * HD / 4, F4 = HD / 4, GROUPS = ROW ? 8 : 1;
    __shared__ unsigned long long red[2 * 2 * HD / 32];
    __shared__ float4 part[GROUPS][F4];
    __shared__ float part_l[GROUPS], top[2 * HD / 32];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t tid = threadIdx.x, f = tid % F4, grp = ROW ? tid / F4 : 0, r = ROW ? blockIdx.x % R : tid / F4, unit = ROW ? blockIdx.x / R : blockIdx.x;
    const uint32_t head = unit % a.c.nkv, rest = unit / a.c.nkv, s = rest / a.tiles;
    unsigned long long ahead, all;
    dealt_sums<R>(a, s, &ahead, &all, red);
    const Dealt d = dealt_of<R>(a, s);
    Seq seq;
    if (d.blocks == 0 || !sequence(a.sq, s, &seq, a.status)) return;
    const uint32_t n = dealt_ctas(all, ctas), rows = seq.count * a.G;
    for (uint32_t tile = rest % a.tiles; tile < d.tiles; tile += a.tiles) {
        const uint32_t row = tile * R + r;
        const unsigned long long from = ahead + ((unsigned long long)tile * a.c.nkv + head) * d.blocks, last = from + d.blocks - 1;
        const uint32_t i0 = (uint32_t)(((from + 1) * n - 1) / all), i1 = (uint32_t)(((last + 1) * n - 1) / all);  // CTA i has all i / n .. all (i + 1) / n, rounded down
        if (i0 == i1 || (ROW && row >= rows)) continue;
        auto place = [&](uint32_t i) { return a.work + (size_t)(2 * i + (all * i / n > from ? 0 : 1)) * DEALT_FLOAT4<HD>; };
        float M = -INFINITY;
        if (ROW) {
            for (uint32_t i = i0 + tid; i <= i1; i += 2 * HD) M = fmaxf(M, __ldcg(place(i) + ITEMS + r).x);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
            if ((tid & 31) == 0) top[tid >> 5] = M;
            __syncthreads();
            for (int w = 0; w < 2 * HD / 32; w++) M = fmaxf(M, top[w]);
        } else {
            for (uint32_t i = i0; i <= i1; i++) M = fmaxf(M, __ldcg(place(i) + ITEMS + r).x);
        }
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float den = 0.0f;
#pragma unroll 4
        for (uint32_t i = i0 + grp; i <= i1; i += GROUPS) {
            const float4 x = __ldcg(place(i) + r * F4 + f), ml = __ldcg(place(i) + ITEMS + r);
            const float k = weight_of(ml.x, M);
            v.x = fmaf(k, x.x, v.x), v.y = fmaf(k, x.y, v.y), v.z = fmaf(k, x.z, v.z), v.w = fmaf(k, x.w, v.w);
            den = fmaf(k, ml.y, den);
        }
        if (ROW) {
            part[grp][f] = v;
            if (f == 0) part_l[grp] = den;
            __syncthreads();
        }
        if (grp == 0 && row < rows) {
            if (ROW) {
#pragma unroll
                for (int k = 1; k < GROUPS; k++) {
                    const float4 x = part[k][f];
                    v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
                    den += part_l[k];
                }
            }
            const float inv = den > 0.0f || den != den ? SUM_UP / den : 0.0f;
            T* const to = (T*)a.out + (size_t)(seq.r0 + row / a.G) * a.out_stride + (size_t)(head * a.G + row % a.G) * HD + f * 4;
            store4<T>(to, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv), a.aligned);
        }
        if (ROW) __syncthreads();
    }
}

template <int HD, int TERMS, bool SPECIAL, typename T>
cudaError_t attend_p(AkArgs& a, uint32_t units_per_tile, uint64_t& launched, cudaStream_t st, bool pdl) {
    using L = AkShared<HD, TERMS>;
    constexpr uint32_t R = TERMS == 2 ? 8 : 16;
    auto kern = attend_kv8_kernel<HD, TERMS, T, SPECIAL, false>;
    const size_t rows = (size_t)a.sq.max_rows * a.G;
    size_t tiles = (rows + R - 1) / R;
    const size_t most = 0x7fffffffu / ((size_t)units_per_tile * 16);
    if (most == 0) return cudaErrorInvalidValue;
    if (tiles > most) tiles = most;
    a.tiles = (uint32_t)tiles;
    const size_t units = tiles * units_per_tile;
    // CTAs of a cluster: as long as all of them fit the chip at two an SM (fourteen clusters of sixteen, 36 of eight) and a warp has two blocks.
    uint32_t C = 1;
    const size_t blocks = a.window && !a.prefix ? std::min<size_t>(a.sq.max_blocks, ((size_t)a.window + a.sq.max_rows) / KV8_BLOCK + 2) : a.sq.max_blocks;
    while (C < 16 && units * C * 2 <= (C == 8 ? 224 : 288) && blocks >= 2 * C * 2 * AK_WARPS) C *= 2;
    if constexpr (TERMS == 2) {
        // Dealt out where that saves a warp six blocks, one behind the other, of what it has otherwise (a launch more, and finding out what is whose, take as long; lengths
        // that differ are put at a quarter off the longest). us, cluster / dealt: one token of 32 heads of 8 KV heads over 8192, 32768 and 131071 keys 15.3 / 18.6,
        // 35.7 / 27.0, 121 / 56; 16 sequences of up to 2000 and 8000 keys 19 / 25, 57 / 40; 64 of up to 4096 75.6 / 70; 256 of up to 2000 127 / 145.
        const double mine = std::max(1.0, (double)units * C / DEALT_CTAS) * blocks / (C * AK_WARPS), dealt_out = 0.75 * units * blocks / (DEALT_CTAS * AK_WARPS) + 6;
        if (a.work && units <= 2 * DEALT_CTAS && mine >= dealt_out) {
            auto dealt = attend_kv8_kernel<HD, TERMS, T, SPECIAL, true>;
            if (cudaError_t e = ensure_dynamic_smem((const void*)dealt, L::BYTES, 0); e != cudaSuccess) return e;
            if (cudaError_t e = launch_k(dealt, dim3(DEALT_CTAS), dim3(AK_THREADS), L::BYTES, st, pdl, a); e != cudaSuccess) return e;
            launched++;
            if (units <= 64) return launch_k(attend_kv8_join<HD, true, T>, dim3((unsigned)units * 8), dim3(2 * HD), 0, st, true, a, DEALT_CTAS);
            return launch_k(attend_kv8_join<HD, false, T>, dim3((unsigned)units), dim3(2 * HD), 0, st, true, a, DEALT_CTAS);
        }
    }
    if (cudaError_t e = ensure_dynamic_smem((const void*)kern, L::BYTES, 0); e != cudaSuccess) return e;
    if (cudaError_t e = cudaFuncSetAttribute((const void*)kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * C));
    cfg.blockDim = dim3(AK_THREADS);
    cfg.dynamicSmemBytes = L::BYTES;
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
template <int HD, int TERMS, typename T>
cudaError_t attend_t(AkArgs& a, uint32_t units_per_tile, uint64_t& launched, cudaStream_t st, bool pdl) {
    return a.cap2 > 0.0f || a.slopes ? attend_p<HD, TERMS, true, T>(a, units_per_tile, launched, st, pdl) : attend_p<HD, TERMS, false, T>(a, units_per_tile, launched, st, pdl);
}
template <int HD>
cudaError_t attend_hd(AkArgs& a, int dtype, uint32_t units_per_tile, uint64_t& launched, cudaStream_t st, bool pdl) {
    const bool few = (size_t)a.sq.max_rows * a.G <= 8;
    switch (dtype) {
        case B2_F32: return attend_t<HD, 2, float>(a, units_per_tile, launched, st, pdl);
        case B2_F16: return few ? attend_t<HD, 2, __half>(a, units_per_tile, launched, st, pdl) : attend_t<HD, 1, __half>(a, units_per_tile, launched, st, pdl);
        case B2_BF16: return few ? attend_t<HD, 2, __nv_bfloat16>(a, units_per_tile, launched, st, pdl) : attend_t<HD, 1, __nv_bfloat16>(a, units_per_tile, launched, st, pdl);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

size_t attend_kv8_work_bytes(uint32_t hd) { return (size_t)DEALT_CTAS * 2 * (hd == 64 ? DEALT_FLOAT4<64> : DEALT_FLOAT4<128>) * 16; }

cudaError_t launch_attend_kv8(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& p, const void* q, size_t q_stride, void* out, size_t out_stride, int dtype,
                              uint32_t* status, uint64_t& launched, cudaStream_t st, bool pdl) {
    if (!kv8_supports(c.nkv, c.hd) || p.nh == 0 || p.nh % c.nkv) return cudaErrorInvalidValue;
    if (s.n_seqs == 0 || s.n_rows == 0 || s.max_rows == 0) return cudaSuccess;
    // Many rows go to the form on tcgen05, from 64 of a KV head and sequence on.
    // mma.sync / tcgen05, us, 4 heads a KV head, 8 KV heads of 128, one sequence behind 4096 keys, eight behind 1024, 32 behind 512: 32 rows 14.2 / 17.7, 13.7 / 15.4, 22.9 / 28.6; 64 rows
    // 14.9 / 18.3, 17.3 / 15.7, 29.0 / 25.8; 128 rows 19.8 / 19.5, 21.7 / 19.0, 50.7 / 29.9; 512 rows 50.5 / 30.5, 64.8 / 26.7, 167 / 52. (One threshold for all numbers of sequences: the
    // hint of a call's longest sequence changes its bits at one place only.)
    launched++;
    if ((dtype != B2_F32 || p.halves) && (size_t)s.max_rows * (p.nh / c.nkv) >= 64 && attend_kv8_rows_supports(c, s, p.nh))
        return launch_attend_kv8_rows(c, s, p, q, q_stride, out, out_stride, dtype, status, st, pdl);
    AkArgs a{};
    a.c = c;
    a.sq = s;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.G = p.nh / c.nkv;
    a.window = p.window <= 0x7fffffffu ? p.window : 0;  // (positions are below 2^31)
    a.c2 = p.scale * 1.44269504f;
    a.cap2 = p.cap * 1.44269504f;
    a.cap_in = p.cap > 0.0f ? 2.0f / p.cap : 0.0f;
    a.slopes = p.slopes;
    a.prefix = p.prefix;
    a.status = status;
    a.work = (float4*)p.work;
    const size_t esz = dtype == B2_F32 ? 4 : 2, unit = 4 * esz;
    a.aligned = (((uintptr_t)q | (uintptr_t)out | q_stride * esz | out_stride * esz) & (unit - 1)) == 0;
    const size_t per_tile = (size_t)s.n_seqs * c.nkv;
    if (per_tile > 0x7fffffffu / 16) return cudaErrorInvalidValue;
    return c.hd == 64 ? attend_hd<64>(a, dtype, (uint32_t)per_tile, launched, st, pdl) : attend_hd<128>(a, dtype, (uint32_t)per_tile, launched, st, pdl);
}

}  // namespace b2
