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
constexpr float P_BITS = 14.0f;  // probabilities are held 2^14 times as large: what is below 2^-28 of a row's largest loses bits, not before

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
    uint32_t* status;
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
    const float2 f = __half22float2(*(const __half2*)&hi);
    return pack(a - f.x, b - f.y);
}
// cap tanh(x / cap), x and the result in powers of two. Near zero by tanh's Taylor series (1 - 2 / (e^2z + 1) would lose bits there).
__device__ __forceinline__ float capped(float x, float cap2, float cap_in) {
    const float z = 0.5f * 0.69314718f * (x * cap_in), z2 = z * z;
    const float series = z * fmaf(z2, fmaf(z2, fmaf(z2, fmaf(z2, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    const float far = 1.0f - __fdividef(2.0f, 1.0f + ex2(x * cap_in));
    return cap2 * (fabsf(z) < 0.3f ? series : far);
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
__device__ __forceinline__ float peer_f(const void* p, uint32_t cta) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer(p, cta)) : "memory");
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

// A CTA's grid index: (unit of work, CTA of the cluster); a unit: (sequence, tile of rows from the last on, KV head).
template <int HD, int TERMS, typename T>
__global__ void __launch_bounds__(AK_THREADS, TERMS == 2 ? 3 : 2) attend_kv8_kernel(const AkArgs a) {
    using L = AkShared<HD, TERMS>;
    constexpr int R = TERMS == 2 ? 8 : 16, RG = TERMS == 2 ? 1 : 2;  // rows of a tile; a lane's rows
    constexpr int KS = HD / 16, NT = HD / 8, QD = HD / 4, S = L::STAGES;
    extern __shared__ __align__(128) uint8_t smem[];
    pdl_launch_dependents();
    const uint32_t C = cluster_size(), cta = cluster_rank();
    const uint32_t work = blockIdx.x / C, head = work % a.c.nkv, rest = work / a.c.nkv, first_tile = a.tiles - 1 - rest % a.tiles, s = rest / a.tiles;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint8_t* const ring = smem + warp * L::RING;
    uint64_t* const bars = (uint64_t*)(smem + L::BARS) + warp * S;
    float* const sum_s = (float*)smem;  // the CTA's sums, where the first warp's were
    float* const m_s = (float*)(smem + L::ML);
    float* const l_s = m_s + 16;
    float* const wm = l_s + 16;                 // [warp][16]
    float* const wl = wm + AK_WARPS * 16;
    if (lane == 0) {
        for (int i = 0; i < S; i++) bar_init(&bars[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    pdl_wait();
    Seq seq;
    if (!sequence(a.sq, s, &seq, a.status)) return;  // (the same in every CTA of the cluster)
    const uint32_t rows = seq.count * a.G, len = seq.start + seq.count;
    const uint32_t prefix = a.prefix ? (uint32_t)min(max(a.prefix[s], 0), (int)len) : 0;
    const uint32_t NW = C * AK_WARPS, gw = cta * AK_WARPS + warp;
    uint32_t slot = 0, phase = 0;
    bool ok = true;

    for (uint32_t tile = first_tile; (size_t)tile * R < rows; tile += a.tiles) {
        const uint32_t row0 = tile * R;
        const uint32_t p_first = seq.start + row0 / a.G, p_last = seq.start + min(row0 + R - 1, rows - 1) / a.G;
        const uint32_t k_end = max(p_last + 1, prefix);                                                // keys below are seen by some row
        const uint32_t k_lo = a.window && p_first + 1 > a.window ? p_first + 1 - a.window : 0;         // keys from here on
        const uint32_t in_lo = a.window && p_last + 1 > a.window ? p_last + 1 - a.window : 0;          // keys from here to in_end are seen by every row
        const uint32_t in_end = max(p_first + 1, prefix);
        const uint32_t b_beg = k_lo / KV8_BLOCK, b_end = (k_end + KV8_BLOCK - 1) / KV8_BLOCK;

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
            slope[i] = a.slopes ? a.slopes[h] * 1.44269504f : 0.0f;
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
            const float k_scale = __uint_as_float(hd.x), v_scale = __uint_as_float(hd.z);
            const uint32_t bad = hd.y | hd.w;
            float sc[RG][8];  // [row][key 2 t + e of tile j]: 2 j + e
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int hf = 0; hf < KS / 4; hf++) {
                    const uint4 w = *(const uint4*)(unit + KV8_HEADER + j * (8 * HD) + hf * 512 + lane * 16);
                    mma16816(d0, qa[4 * hf], low_half(w.x), high_half(w.x));
                    mma16816(d1, qa[4 * hf + 1], low_half(w.y), high_half(w.y));
                    mma16816(d0, qa[4 * hf + 2], low_half(w.z), high_half(w.z));
                    mma16816(d1, qa[4 * hf + 3], low_half(w.w), high_half(w.w));
                }
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    if constexpr (TERMS == 2) {
                        sc[0][2 * j + e] = (d0[e] + d1[e]) + (d0[2 + e] + d1[2 + e]);
                    } else {
                        sc[0][2 * j + e] = d0[e] + d1[e];
                        sc[RG - 1][2 * j + e] = d0[2 + e] + d1[2 + e];
                    }
                }
            }
            const bool whole = key0 >= in_lo && key0 + KV8_BLOCK <= in_end && bad == 0;  // every row sees every key
            uint32_t ph[RG][4], pl[4];  // probabilities of keys 4 t + 2 j .. : tile j's two
            float shrink[RG];
            bool grown = false;
#pragma unroll
            for (int i = 0; i < RG; i++) {
                const float f = qf[i] * k_scale;
                float mx = -INFINITY;
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    const uint32_t key = key0 + 16 * (x >> 2) + 4 * t + (x & 3);
                    float y = sc[i][x] * f;
                    if (a.cap2 > 0.0f) y = capped(y, a.cap2, a.cap_in);
                    if (a.slopes) y = fmaf(slope[i], (float)(int)(key - pos[i]), y);
                    if (!whole) {
                        const bool see = key < len && (key <= pos[i] || key < prefix) && (a.window == 0 || (int)(pos[i] - key) < (int)a.window);
                        if ((bad >> (key - key0)) & 1) y = NAN;
                        if (!see) y = -INFINITY;
                    }
                    sc[i][x] = y;
                    mx = fmaxf(mx, y);
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.0f : mn;
                shrink[i] = ex2(m[i] - base);
                grown = grown || mn > m[i];
                m[i] = mn;
                float add = 0.0f;
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    sc[i][x] = ex2(sc[i][x] - base + P_BITS);
                    add += sc[i][x];
                }
                l[i] = fmaf(l[i], shrink[i], add);
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
                    for (int e = 0; e < 2 * RG; e++) o[n][e] *= shrink[e >> 1];
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
                float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816(d0, pa[0], low_half(w.x), high_half(w.x));
                mma16816(d1, pa[0], low_half(w.z), high_half(w.z));
                mma16816(d0, pa[1], low_half(w.y), high_half(w.y));
                mma16816(d1, pa[1], low_half(w.w), high_half(w.w));
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    if constexpr (TERMS == 2) {
                        o[n][e] = fmaf(d0[e] + d0[2 + e], v_scale, o[n][e]);
                        o[n + 1][e] = fmaf(d1[e] + d1[2 + e], v_scale, o[n + 1][e]);
                    } else {
                        o[n][e] = fmaf(d0[e], v_scale, o[n][e]);
                        o[n][2 * RG - 2 + e] = fmaf(d0[2 + e], v_scale, o[n][2 * RG - 2 + e]);
                        o[n + 1][e] = fmaf(d1[e], v_scale, o[n + 1][e]);
                        o[n + 1][2 * RG - 2 + e] = fmaf(d1[2 + e], v_scale, o[n + 1][2 * RG - 2 + e]);
                    }
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
            const float inv = den > 0.0f || den != den ? 1.0f / den : 0.0f;  // (a row that sees nothing: zeros)
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
            if (C == 1) {
                finish(item, v, den);
            } else {
                ((float4*)sum_s)[item] = v;
                if (item % (HD / 4) == 0) {
                    m_s[r] = M;
                    l_s[r] = den;
                }
            }
        }
        if (C > 1) {
            cluster_sync();
            for (int item = (int)cta * AK_THREADS + tid; item < ITEMS; item += (int)C * AK_THREADS) {
                const int r = item / (HD / 4);
                float M = -INFINITY, den = 0.0f;
                for (uint32_t k = 0; k < C; k++) M = fmaxf(M, peer_f(m_s + r, k));
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                for (uint32_t k = 0; k < C; k++) {
                    const float w = weight_of(peer_f(m_s + r, k), M);
                    const float4 x = peer_f4((const float4*)sum_s + item, k);
                    v.x = fmaf(w, x.x, v.x), v.y = fmaf(w, x.y, v.y), v.z = fmaf(w, x.z, v.z), v.w = fmaf(w, x.w, v.w);
                    den = fmaf(w, peer_f(l_s + r, k), den);
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
    }
}

template <int HD, int TERMS, typename T>
cudaError_t attend_t(AkArgs& a, uint32_t units_per_tile, cudaStream_t st, bool pdl) {
    using L = AkShared<HD, TERMS>;
    constexpr uint32_t R = TERMS == 2 ? 8 : 16;
    auto kern = attend_kv8_kernel<HD, TERMS, T>;
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
template <int HD>
cudaError_t attend_hd(AkArgs& a, int dtype, uint32_t units_per_tile, cudaStream_t st, bool pdl) {
    const bool few = (size_t)a.sq.max_rows * a.G <= 8;
    switch (dtype) {
        case B2_F32: return attend_t<HD, 2, float>(a, units_per_tile, st, pdl);
        case B2_F16: return few ? attend_t<HD, 2, __half>(a, units_per_tile, st, pdl) : attend_t<HD, 1, __half>(a, units_per_tile, st, pdl);
        case B2_BF16: return few ? attend_t<HD, 2, __nv_bfloat16>(a, units_per_tile, st, pdl) : attend_t<HD, 1, __nv_bfloat16>(a, units_per_tile, st, pdl);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_attend_kv8(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& p, const void* q, size_t q_stride, void* out, size_t out_stride, int dtype,
                              uint32_t* status, cudaStream_t st, bool pdl) {
    if (!kv8_supports(c.nkv, c.hd) || p.nh == 0 || p.nh % c.nkv) return cudaErrorInvalidValue;
    if (s.n_seqs == 0 || s.n_rows == 0 || s.max_rows == 0) return cudaSuccess;
    // Many rows go to the form on tcgen05, from 64 of a KV head and sequence on. mma.sync / tcgen05, us, 4 heads a KV head, 8 KV heads of 128, one sequence behind
    // 4096 keys, eight behind 1024, 32 behind 512: 64 rows 18.1 / 19.7, 22.1 / 18.3, 35.5 / 31.2; 128 rows 26.3 / 21.4, 28.2 / 21.9, 62.8 / 36.1; 512 rows 76 / 30, 84 / 31.
    if ((dtype != B2_F32 || p.halves) && (size_t)s.max_rows * (p.nh / c.nkv) >= 64)
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
    const size_t esz = dtype == B2_F32 ? 4 : 2, unit = 4 * esz;
    a.aligned = (((uintptr_t)q | (uintptr_t)out | q_stride * esz | out_stride * esz) & (unit - 1)) == 0;
    const size_t per_tile = (size_t)s.n_seqs * c.nkv;
    if (per_tile > 0x7fffffffu / 16) return cudaErrorInvalidValue;
    return c.hd == 64 ? attend_hd<64>(a, dtype, (uint32_t)per_tile, st, pdl) : attend_hd<128>(a, dtype, (uint32_t)per_tile, st, pdl);
}

}  // namespace b2
