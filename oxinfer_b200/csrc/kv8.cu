// The 8-bit cache (kv8.cuh): rows of keys and values into it, and the values that it holds out of it. The reference's caches are f32
// (LayerCache, src/model.rs); this one holds a quarter of their bytes, so that attention reads a quarter.
//
// append: scale = 2^e, e the smallest with largest magnitude <= 127 * 2^e over the block's new rows (not below 2^-100), and not below the scale of the
// rows of the block that stay; q = round half to even (x / scale), exact but for that rounding (at the scale 2^122 at most 63, so that the value is finite). Rows that stay are brought to a larger scale the same way.
// A row with a value that is not finite is marked, and counts as NaN: it does not enter the scale, and the block's other rows are as they would be without it.
#include "kv8.cuh"

#include <cfloat>

#include "pdl.cuh"

namespace b2 {

using namespace kv8;

namespace {

constexpr int KV_THREADS = 256;  // eight threads a token: thread i has dimensions 4 i .. 4 i + 3 and every 32nd behind them

// e of the largest magnitude: mantissas up to 127 / 64 fit 127 * 2^(exponent - 6).
__device__ __forceinline__ int scale_exponent(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int x = (int)(b >> 23) - 127;
    return max((b & 0x7fffffu) <= 0x7e0000u ? x - 6 : x - 5, -100);
}
// `most`: 127, but 63 at the largest scale, 2^122, where 64 would no longer be a finite value.
__device__ __forceinline__ uint32_t to_byte(float q, float most) { return (uint32_t)((int)fminf(fmaxf(rintf(q), -most), most) + 128); }

template <int HD, typename T>
__global__ void __launch_bounds__(KV_THREADS) append_kernel(Kv8Cache c, Kv8Seqs sq, Kv8Rows x, uint32_t tiles, int keep_behind, int aligned, uint32_t* status) {
    constexpr int C = HD / 32, UNIT = (int)unit_bytes(HD);
    __shared__ __align__(16) uint8_t image[2 * KV8_BLOCK * HD];
    __shared__ float warp_max[2][KV_THREADS / 32];
    __shared__ uint32_t warp_bad[2][KV_THREADS / 32];
    pdl_launch_dependents();
    const int tid = threadIdx.x, r = tid >> 3, i4 = (tid & 7) * 4, warp = tid >> 5, lane = tid & 31;
    const uint32_t head = blockIdx.x % c.nkv, rest = blockIdx.x / c.nkv, tile = rest % tiles, s = rest / tiles;
    pdl_wait();
    Seq seq;
    if (!sequence(sq, s, &seq, status) || seq.count == 0) return;
    const uint32_t end = seq.start + seq.count, b_end = (end - 1) / KV8_BLOCK + 1;
    for (uint32_t b = seq.start / KV8_BLOCK + tile; b < b_end; b += tiles) {
        const int id = block_of(c, sq, s, b, status);
        if (id < 0) continue;
        uint8_t* const unit = c.units + ((size_t)id * c.nkv + head) * UNIT;
        const int base = (int)(b * KV8_BLOCK);  // (positions are below 2^31)
        const int lo = max((int)seq.start - base, 0), hi = min((int)end - base, (int)KV8_BLOCK);
        const bool kept = lo > 0 || (keep_behind && hi < (int)KV8_BLOCK), is_new = r >= lo && r < hi, stays = !is_new && (r < lo || keep_behind);
        Header old = *(const Header*)unit;
        float v[2][C][4];
        float top[2] = {0.0f, 0.0f};
        bool fine[2] = {true, true};
#pragma unroll
        for (int kind = 0; kind < 2; kind++) {
            const T* const row = (const T*)(kind ? x.v : x.k) + (size_t)(is_new ? seq.r0 + (uint32_t)(base + r) - seq.start : 0u) * x.rs + (size_t)head * x.hs;
#pragma unroll
            for (int j = 0; j < C; j++) {
                if (is_new) {
                    load4(v[kind][j], row + i4 + 32 * j, aligned);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) v[kind][j][e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float a = fabsf(v[kind][j][e]);
                    fine[kind] = fine[kind] && a <= FLT_MAX;
                    top[kind] = fmaxf(top[kind], a);
                }
            }
        }
#pragma unroll
        for (int kind = 0; kind < 2; kind++) {
            const uint32_t odd = __ballot_sync(0xffffffffu, !fine[kind]);  // a byte for each of the warp's four rows
            uint32_t bad = 0;
#pragma unroll
            for (int w = 0; w < 4; w++) bad |= ((odd >> (8 * w)) & 0xffu) ? 1u << w : 0u;
            fine[kind] = !((bad >> (lane >> 3)) & 1u);
            float m = fine[kind] ? top[kind] : 0.0f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (lane == 0) {
                warp_max[kind][warp] = m;
                warp_bad[kind][warp] = bad << (4 * warp);
            }
        }
        __syncthreads();  // (the old header has been read by everyone, too)
        const uint32_t staying = ~(uint32_t)((((1ull << hi) - 1) >> lo) << lo) & (keep_behind ? 0xffffffffu : (uint32_t)((1ull << lo) - 1));
        float scale[2], shrink[2];
        uint32_t bad_bits[2];
        bool grows = false;
#pragma unroll
        for (int kind = 0; kind < 2; kind++) {
            float m = 0.0f;
            uint32_t bad = kept ? (kind ? old.v_bad : old.k_bad) & staying : 0u;
#pragma unroll
            for (int w = 0; w < KV_THREADS / 32; w++) {
                m = fmaxf(m, warp_max[kind][w]);
                bad |= warp_bad[kind][w];
            }
            bad_bits[kind] = bad;
            const float was = kept ? (kind ? old.v_scale : old.k_scale) : 0.0f;
            scale[kind] = fmaxf(pow2(scale_exponent(m)), was);
            shrink[kind] = was / scale[kind];  // (a power of two, 0 where nothing was written yet)
            grows = grows || (kept && was < scale[kind]);
        }
        // Whole blocks and those whose rows change leave as one image, 16 bytes a thread; a few rows (a decoding step) byte by byte, in place.
        const bool whole = grows || hi - lo >= 8;
        if (whole && kept) {
            for (int o = tid; o < (int)(2 * KV8_BLOCK * HD / 16); o += KV_THREADS) ((uint4*)image)[o] = ((const uint4*)(unit + KV8_HEADER))[o];
            __syncthreads();
        }
        if (whole || is_new) {
            uint8_t* const to = whole ? image : unit + KV8_HEADER;
#pragma unroll
            for (int kind = 0; kind < 2; kind++) {
                const float inv = 1.0f / scale[kind], most = inv == 0x1p-122f ? 63.0f : 127.0f;
#pragma unroll
                for (int j = 0; j < C; j++) {
                    const uint32_t d = i4 + 32 * j;
                    uint32_t q[4];
                    if (is_new) {
#pragma unroll
                        for (int e = 0; e < 4; e++) q[e] = fine[kind] ? to_byte(v[kind][j][e] * inv, most) : 128u;
                    } else if (stays && kept) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t at = kind ? KV8_BLOCK * HD + value_at(r, d + e) : key_at<HD>(r, d) + e;
                            q[e] = to_byte((float)((int)image[at] - 128) * shrink[kind], most);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) q[e] = 128u;
                    }
                    if (kind == 0) {
                        *(uint32_t*)(to + key_at<HD>(r, d)) = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) to[KV8_BLOCK * HD + value_at(r, d + e)] = (uint8_t)q[e];
                    }
                }
            }
        }
        if (tid == 0) *(Header*)unit = Header{scale[0], bad_bits[0], scale[1], bad_bits[1], {0, 0, 0, 0}};
        __syncthreads();
        if (whole)
            for (int o = tid; o < (int)(2 * KV8_BLOCK * HD / 16); o += KV_THREADS) ((uint4*)(unit + KV8_HEADER))[o] = ((const uint4*)image)[o];
        __syncthreads();
    }
}

template <int HD>
__global__ void __launch_bounds__(KV_THREADS) read_kernel(Kv8Cache c, Kv8Seqs sq, float* __restrict__ k, float* __restrict__ v, uint32_t tiles, uint32_t* status) {
    constexpr int C = HD / 32, UNIT = (int)unit_bytes(HD);
    __shared__ __align__(16) uint8_t image[UNIT];
    const int tid = threadIdx.x, r = tid >> 3, i4 = (tid & 7) * 4;
    const uint32_t head = blockIdx.x % c.nkv, rest = blockIdx.x / c.nkv, tile = rest % tiles, s = rest / tiles;
    Seq seq;
    if (!sequence(sq, s, &seq, status) || seq.count == 0) return;
    const uint32_t end = seq.start + seq.count, b_end = (end - 1) / KV8_BLOCK + 1;
    for (uint32_t b = seq.start / KV8_BLOCK + tile; b < b_end; b += tiles) {
        const int id = block_of(c, sq, s, b, status);
        if (id < 0) continue;
        const uint8_t* const unit = c.units + ((size_t)id * c.nkv + head) * UNIT;
        __syncthreads();
        for (int o = tid; o < UNIT / 16; o += KV_THREADS) ((uint4*)image)[o] = ((const uint4*)unit)[o];
        __syncthreads();
        const uint32_t pos = b * KV8_BLOCK + r;
        if (pos < seq.start || pos >= end) continue;
        const Header h = *(const Header*)image;
        const float ks = (h.k_bad >> r) & 1 ? NAN : h.k_scale, vs = (h.v_bad >> r) & 1 ? NAN : h.v_scale;
        const size_t to = ((size_t)(seq.r0 + (pos - seq.start)) * c.nkv + head) * HD;
#pragma unroll
        for (int j = 0; j < C; j++) {
            const uint32_t d = i4 + 32 * j;
            const uint8_t* const kb = image + KV8_HEADER + key_at<HD>(r, d);
            const uint8_t* const vb = image + KV8_HEADER + KV8_BLOCK * HD;
            float a[4], e[4];
#pragma unroll
            for (int m = 0; m < 4; m++) {
                a[m] = (float)((int)kb[m] - 128) * ks;
                e[m] = (float)((int)vb[value_at(r, d + m)] - 128) * vs;
            }
            *(float4*)(k + to + d) = make_float4(a[0], a[1], a[2], a[3]);
            *(float4*)(v + to + d) = make_float4(e[0], e[1], e[2], e[3]);
        }
    }
}

// Blocks that the rows of one sequence may reach into.
uint32_t tiles_of(const Kv8Seqs& s) { return (uint32_t)(((size_t)s.max_rows + 2 * KV8_BLOCK - 2) / KV8_BLOCK); }

template <int HD, typename T>
cudaError_t append_t(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Rows& x, bool keep_behind, uint32_t* status, cudaStream_t st, bool pdl) {
    uint32_t tiles = tiles_of(s);
    const size_t most = 0x7fffffffu / ((size_t)c.nkv * s.n_seqs);
    if (most == 0) return cudaErrorInvalidValue;
    if (tiles > most) tiles = (uint32_t)most;
    const size_t unit = 4 * sizeof(T);
    const int aligned = (((uintptr_t)x.k | (uintptr_t)x.v | x.rs * sizeof(T) | x.hs * sizeof(T)) & (unit - 1)) == 0;
    return launch_k(append_kernel<HD, T>, dim3(tiles * c.nkv * s.n_seqs), dim3(KV_THREADS), 0, st, pdl, c, s, x, tiles, keep_behind ? 1 : 0, aligned, status);
}
template <int HD>
cudaError_t append_hd(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Rows& x, bool keep_behind, uint32_t* status, cudaStream_t st, bool pdl) {
    switch (x.dtype) {
        case B2_F32: return append_t<HD, float>(c, s, x, keep_behind, status, st, pdl);
        case B2_BF16: return append_t<HD, __nv_bfloat16>(c, s, x, keep_behind, status, st, pdl);
        case B2_F16: return append_t<HD, __half>(c, s, x, keep_behind, status, st, pdl);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

bool kv8_supports(uint32_t nkv, uint32_t hd) { return nkv > 0 && nkv <= 4096 && (hd == 64 || hd == 128); }
size_t kv8_bytes(uint32_t nkv, uint32_t hd, uint32_t n_blocks) { return (size_t)n_blocks * nkv * unit_bytes(hd); }

cudaError_t launch_kv8_append(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Rows& x, bool keep_behind, uint32_t* status, cudaStream_t st, bool pdl) {
    if (!kv8_supports(c.nkv, c.hd)) return cudaErrorInvalidValue;
    if (s.n_seqs == 0 || s.n_rows == 0 || s.max_rows == 0) return cudaSuccess;
    return c.hd == 64 ? append_hd<64>(c, s, x, keep_behind, status, st, pdl) : append_hd<128>(c, s, x, keep_behind, status, st, pdl);
}

cudaError_t launch_kv8_read(const Kv8Cache& c, const Kv8Seqs& s, float* k, float* v, uint32_t* status, cudaStream_t st) {
    if (!kv8_supports(c.nkv, c.hd)) return cudaErrorInvalidValue;
    if (s.n_seqs == 0 || s.n_rows == 0 || s.max_rows == 0) return cudaSuccess;
    uint32_t tiles = tiles_of(s);
    const size_t most = 0x7fffffffu / ((size_t)c.nkv * s.n_seqs);
    if (most == 0) return cudaErrorInvalidValue;
    if (tiles > most) tiles = (uint32_t)most;
    if (c.hd == 64) read_kernel<64><<<tiles * c.nkv * s.n_seqs, KV_THREADS, 0, st>>>(c, s, k, v, tiles, status);
    else read_kernel<128><<<tiles * c.nkv * s.n_seqs, KV_THREADS, 0, st>>>(c, s, k, v, tiles, status);
    return cudaGetLastError();
}

}  // namespace b2
