// The 8-bit cache (kv8.cuh): rows of keys and values into it, and the values that it holds out of it. The reference's caches are f32
// (LayerCache, src/model.rs); this one holds a quarter of their bytes, so that attention reads a quarter.
//
// append: scale = 2^e, e the smallest with largest magnitude <= 127 * 2^e over the block's new rows (not below 2^-100), and not below the scale of the
// rows of the block that stay; q = round half to even (x / scale), exact but for that rounding (at the scale 2^122 at most 63, so that the value is finite). Rows that stay are brought to a larger scale the same way.
// What bounds it (times of replays with warm caches): a prompt of 8192 rows of 8 KV heads of 128 the issue slots beside HBM, f32 rows appended in 15.1 us (84 MB, 5.6 TB/s), bf16 in 12.7 (50 MB, 4 TB/s), read back in 14.2
// (84 MB, 5.9 TB/s); a step of 64 sequences a launch and three dependent reads, 2.8 and 2.3 us.
// A row with a value that is not finite is marked, and counts as NaN: it does not enter the scale, and the block's other rows are as they would be without it.
#include "kv8.cuh"

#include <algorithm>
#include <cfloat>

#include "attend_core.cuh"
#include "pdl.cuh"

namespace b2 {

using namespace kv8;

namespace {

constexpr uint32_t FEW = 4;  // rows of a sequence that a warp a block has
constexpr int KV_CTAS = 4;       // of an SM
constexpr size_t KV_WAVE = 8;    // of a launch over many blocks, which fetch a block's rows while they write the one ahead
constexpr int KV_THREADS = 256;  // eight threads a token

// e of the largest magnitude: mantissas up to 127 / 64 fit 127 * 2^(exponent - 6).
__device__ __forceinline__ int scale_exponent(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int x = (int)(b >> 23) - 127;
    return max((b & 0x7fffffu) <= 0x7e0000u ? x - 6 : x - 5, -100);
}
// `most`: 127, but 63 at the largest scale, 2^122, where 64 would no longer be a finite value.
__device__ __forceinline__ uint32_t to_byte(float q, float most) { return (uint32_t)((int)fminf(fmaxf(rintf(q), -most), most) + 128); }

// Sixteen bytes of a unit's keys or values, from byte `at` on: those of tokens that stay, times `shrink`, rounded.
template <int HD>
__device__ __forceinline__ uint4 requantized(uint4 w, uint32_t at, uint32_t kind, uint32_t staying, float shrink, float most) {
    uint32_t x[4] = {w.x, w.y, w.z, w.w};
    const uint32_t lane = (at & 511) >> 4, n = lane >> 2, j = at / (8 * HD);
    const uint32_t token = 16 * (j >> 1) + 4 * (n >> 1) + 2 * (j & 1) + (n & 1);  // of all sixteen keys
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t y = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t q = (x[i] >> (8 * e)) & 0xffu, tok = kind ? 16 * (i & 1) + 4 * (lane & 3) + e : token;
            y |= ((staying >> tok) & 1 ? to_byte((float)((int)q - 128) * shrink, most) : q) << (8 * e);
        }
        x[i] = y;
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
}
// The rows lo .. hi - 1 of a block that are written, and those that stay.
__device__ __forceinline__ uint32_t rows_between(int lo, int hi) { return (uint32_t)((((1ull << hi) - 1) >> lo) << lo); }
__device__ __forceinline__ uint32_t rows_staying(int lo, int hi, int keep_behind) { return ~rows_between(lo, hi) & (keep_behind ? 0xffffffffu : rows_between(0, lo)); }

// The largest magnitude of a word's values, by its bits as f32 (infinities and NaN above all others), so far.
template <typename T>
__device__ __forceinline__ uint32_t top_of(uint32_t top, uint32_t word) {
    if constexpr (sizeof(T) == 4) return max(top, word & 0x7fffffffu);
    else return __vmaxu2(top, word & 0x7fff7fffu);  // (two 16-bit values, as they are)
}
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint32_t top) {
    if constexpr (sizeof(T) == 4) return top;
    const unsigned short m = (unsigned short)max(top & 0xffffu, top >> 16);
    return __float_as_uint(to_f32<T>(*(const T*)&m));
}

// Grid: (sequence, block of the rows', KV head), a CTA each: the unit's image in shared memory, then out of it 16 bytes a thread at a time. A thread has eight
// dimensions (and eight of the other half of 128) of a token's keys and values. 8192 rows of 8 KV heads of 128, us, f32 and bf16: keys and values
// a CTA each, four dimensions at a time and a barrier more a block 19.2 and 19.3, eight dimensions and six CTAs an SM 17.9 and 16.1, both kinds by one CTA 15.1 and 12.7 (that
// halves what is done once a block; issue slots bound it, 69 % of them).
template <int HD, typename T>
__global__ void __launch_bounds__(KV_THREADS, KV_CTAS) append_kernel(Kv8Cache c, Kv8Seqs sq, Kv8Rows x, uint32_t tiles, int keep_behind, int wide, uint32_t* status) {
    constexpr int J = HD / 64, UNIT = (int)unit_bytes(HD), WARPS = KV_THREADS / 32, IMAGE = (int)KV8_BLOCK * HD, WORDS = IMAGE / 16, V = 16 / (int)sizeof(T), PARTS = 8 / V;
    __shared__ __align__(16) uint8_t images[2][2 * IMAGE];  // keys, then values (in turn: a block's is written while the one ahead's may still be on its way out)
    __shared__ __align__(16) uint32_t warp_top[2][WARPS], warp_bad[2][WARPS];
    pdl_launch_dependents();
    const int tid = threadIdx.x, r = tid >> 3, d8 = (tid & 7) * 8, warp = tid >> 5, lane = tid & 31;
    const uint32_t head = blockIdx.x % c.nkv, rest = blockIdx.x / c.nkv, tile = rest % tiles, s = rest / tiles;
    pdl_wait();
    Seq seq;
    if (!sequence(sq, s, &seq, status) || seq.count == 0) return;
    const uint32_t end = seq.start + seq.count, b_end = (end - 1) / KV8_BLOCK + 1;
    uint32_t b = seq.start / KV8_BLOCK + tile;
    if (b >= b_end) return;
    const size_t from = (size_t)head * x.hs + d8;
    auto rows_of = [&](uint32_t b, int* lo, int* hi) {
        const int base = (int)(b * KV8_BLOCK);  // (positions are below 2^31)
        *lo = max((int)seq.start - base, 0);
        *hi = min((int)end - base, (int)KV8_BLOCK);
    };
    uint4 v[2][J * PARTS];
    int id;
    auto fetch = [&](uint32_t b) {  // a block's rows and its place
        int lo, hi;
        rows_of(b, &lo, &hi);
        const bool is_new = r >= lo && r < hi;
        const size_t row = from + (size_t)(is_new ? seq.r0 + b * KV8_BLOCK + (uint32_t)r - seq.start : 0u) * x.rs;
#pragma unroll
        for (int kind = 0; kind < 2; kind++) {
            const T* const at = (const T*)(kind ? x.v : x.k) + row;
#pragma unroll
            for (int j = 0; j < J * PARTS; j++) v[kind][j] = make_uint4(0, 0, 0, 0);
            if (is_new && wide) {
#pragma unroll
                for (int j = 0; j < J * PARTS; j++) v[kind][j] = *(const uint4*)(at + 64 * (j / PARTS) + V * (j % PARTS));
            } else if (is_new) {
#pragma unroll
                for (int j = 0; j < J * PARTS; j++)
#pragma unroll
                    for (int e = 0; e < V; e++) ((T*)&v[kind][j])[e] = at[64 * (j / PARTS) + V * (j % PARTS) + e];
            }
        }
        id = block_of(c, sq, s, b, status);
    };
    fetch(b);
    for (uint32_t turn = 0; b < b_end; b += tiles) {
        int lo, hi;
        rows_of(b, &lo, &hi);
        const bool is_new = r >= lo && r < hi;
        const uint32_t staying = rows_staying(lo, hi, keep_behind);
        if (id < 0) {
            if (b + tiles < b_end) fetch(b + tiles);
            continue;
        }
        uint8_t* const unit = c.units + ((size_t)id * c.nkv + head) * UNIT;  // (begins with the keys' scale and tokens that are not finite, and the values')
        uint8_t* const image = images[turn ^= 1];
        uint4 old = make_uint4(0, 0, 0, 0);
        if (staying) old = *(const uint4*)unit;
        bool fine[2];
#pragma unroll
        for (int kind = 0; kind < 2; kind++) {
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < J * PARTS; j++) top = top_of<T>(top_of<T>(top_of<T>(top_of<T>(top, v[kind][j].x), v[kind][j].y), v[kind][j].z), v[kind][j].w);
            top = top_bits<T>(top);
            fine[kind] = top < 0x7f800000u;
            const uint32_t odd = __ballot_sync(0xffffffffu, !fine[kind]);  // a byte for each of the warp's four rows
            uint32_t bad = 0;
            if (odd) {
#pragma unroll
                for (int w = 0; w < 4; w++) bad |= ((odd >> (8 * w)) & 0xffu) ? 1u << w : 0u;
                fine[kind] = !((bad >> (lane >> 3)) & 1u);
            }
            const uint32_t m = __reduce_max_sync(0xffffffffu, fine[kind] ? top : 0u);
            if (lane == 0) {
                warp_top[kind][warp] = m;
                warp_bad[kind][warp] = bad << (4 * warp);
            }
        }
        __syncthreads();  // (the old header has been read by everyone, too)
        float was[2] = {__uint_as_float(old.x), __uint_as_float(old.z)}, scale[2], inv[2], most[2];
        uint32_t bad[2] = {old.y & staying, old.w & staying};
#pragma unroll
        for (int kind = 0; kind < 2; kind++) {
            static_assert(WARPS == 8);
            const uint4 t0 = *(const uint4*)warp_top[kind], t1 = *(const uint4*)(warp_top[kind] + 4), b0 = *(const uint4*)warp_bad[kind], b1 = *(const uint4*)(warp_bad[kind] + 4);
            const uint32_t m = max(max(max(t0.x, t0.y), max(t0.z, t0.w)), max(max(t1.x, t1.y), max(t1.z, t1.w)));
            bad[kind] |= b0.x | b0.y | b0.z | b0.w | b1.x | b1.y | b1.z | b1.w;
            scale[kind] = fmaxf(pow2(scale_exponent(__uint_as_float(m))), was[kind]);
            inv[kind] = __uint_as_float((254u << 23) - __float_as_uint(scale[kind]));  // (powers of two)
            most[kind] = inv[kind] == 0x1p-122f ? 63.0f : 127.0f;
        }
        if (hi - lo < (int)KV8_BLOCK) {  // what the image has of other rows
#pragma unroll
            for (int kind = 0; kind < 2; kind++)
                for (int o = tid; o < WORDS; o += KV_THREADS) {
                    uint4 w = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
                    if (staying) {
                        w = ((const uint4*)(unit + KV8_HEADER + kind * IMAGE))[o];
                        if (was[kind] < scale[kind]) w = requantized<HD>(w, 16 * o, kind, staying, was[kind] * inv[kind], most[kind]);
                    }
                    ((uint4*)(image + kind * IMAGE))[o] = w;
                }
            __syncthreads();
        }
        uint32_t w[2][2 * J];  // of four dimensions
#pragma unroll
        for (int kind = 0; kind < 2; kind++)
#pragma unroll
            for (int j = 0; j < 2 * J; j++) {
                const T* const four = (const T*)v[kind] + 4 * j;
                if (!fine[kind]) {
                    w[kind][j] = 0x80808080u;
                } else if (most[kind] == 127.0f) {  // a sum with 1.5 * 2^23 is rounded to a whole number, to even, and its last byte is the byte
                    uint32_t q[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) q[e] = __float_as_uint(fmaf(to_f32<T>(four[e]), inv[kind], 12582912.0f + 128.0f));
                    w[kind][j] = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
                } else {
                    w[kind][j] = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) w[kind][j] |= to_byte(to_f32<T>(four[e]) * inv[kind], most[kind]) << (8 * e);
                }
            }
        if (b + tiles < b_end) fetch(b + tiles);  // (under this block's way out)
#pragma unroll
        for (int j = 0; j < J; j++)
            if (is_new) *(uint2*)(image + key_at<HD>(r, d8 + 64 * j)) = make_uint2(w[0][2 * j], w[0][2 * j + 1]);
        const uint32_t l0 = (lane >> 3) & 1, l1 = lane >> 4, quad = (rows_between(lo, hi) >> (4 * warp)) & 0xfu;  // the warp's four tokens
        if (quad) {
            const uint32_t keep = ~(((quad & 1) | (quad & 2) << 7 | (quad & 4) << 14 | (quad & 8) << 21) * 0xffu);
#pragma unroll
            for (int j = 0; j < 2 * J; j++) {  // four dimensions of a token to four tokens of a dimension, over the lanes of the four tokens
                const uint32_t p = __shfl_xor_sync(0xffffffffu, w[1][j], 8), z = __byte_perm(w[1][j], p, l0 ? 0x3715 : 0x6240);
                const uint32_t p2 = __shfl_xor_sync(0xffffffffu, z, 16), y = __byte_perm(z, p2, l1 ? 0x3276 : 0x5410);
                uint32_t* const to = (uint32_t*)(image + IMAGE + value_at(4 * warp, d8 + 64 * (j >> 1) + 4 * (j & 1) + 2 * l1 + l0));
                *to = keep ? (*to & keep) | (y & ~keep) : y;
            }
        }
        if (tid == 0) *(uint4*)unit = make_uint4(__float_as_uint(scale[0]), bad[0], __float_as_uint(scale[1]), bad[1]);
        __syncthreads();
        for (int o = tid; o < 2 * WORDS; o += KV_THREADS) ((uint4*)(unit + KV8_HEADER))[o] = ((const uint4*)image)[o];
    }
}

// Rows lo .. hi - 1 of a block, of one head and kind, into its unit, by a warp; row lo begins at `from`, and `old` is the unit's scale and tokens that are not finite.
// Bytes are written where they lie. Rows behind the first four are read twice, for the scale and for the bytes.
template <int HD, typename T>
__device__ __forceinline__ void append_rows(uint8_t* unit, uint32_t kind, uint2 old, int lo, int hi, uint32_t staying, const T* from, size_t rs, bool aligned) {
    constexpr int WORDS = (int)KV8_BLOCK * HD / 16, LANES = HD / 4, KEEP = (int)FEW;  // lanes of a row, four dimensions each; rows that are asked for at once
    const int lane = threadIdx.x & 31;
    auto load = [&](float (&v)[4], int r) { load4(v, from + (size_t)(r - lo) * rs + 4 * (lane % LANES), aligned); };
    uint8_t* const bytes = unit + KV8_HEADER + kind * (KV8_BLOCK * HD);
    float kept[KEEP][4];
#pragma unroll
    for (int i = 0; i < KEEP; i++)
        if (lo + i < hi) load(kept[i], lo + i);
    uint32_t top = 0, bad = old.y & staying;
    auto look = [&](const float (&v)[4], int r) {
        const float m = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
        const bool fine = fabsf(v[0]) <= FLT_MAX && fabsf(v[1]) <= FLT_MAX && fabsf(v[2]) <= FLT_MAX && fabsf(v[3]) <= FLT_MAX;
        if (__all_sync(0xffffffffu, fine)) top = max(top, __reduce_max_sync(0xffffffffu, __float_as_uint(m)));
        else bad |= 1u << r;
    };
#pragma unroll
    for (int i = 0; i < KEEP; i++)
        if (lo + i < hi) look(kept[i], lo + i);
    for (int r = lo + KEEP; r < hi; r++) {
        float v[4];
        load(v, r);
        look(v, r);
    }
    const float was = __uint_as_float(old.x), scale = fmaxf(pow2(scale_exponent(__uint_as_float(top))), was);
    const float inv = 1.0f / scale, most = inv == 0x1p-122f ? 63.0f : 127.0f;
    if (staying && was < scale) {
        const float shrink = was * inv;
#pragma unroll 4
        for (int o = lane; o < WORDS; o += 32) ((uint4*)bytes)[o] = requantized<HD>(((const uint4*)bytes)[o], 16 * o, kind, staying, shrink, most);
        __syncwarp();
    }
    auto write = [&](const float (&v)[4], int r) {
        uint32_t q[4];
#pragma unroll
        for (int e = 0; e < 4; e++) q[e] = (bad >> r) & 1 ? 128u : to_byte(v[e] * inv, most);
        if (lane >= LANES) return;
        if (kind == 0) {
            *(uint32_t*)(bytes + key_at<HD>(r, 4 * lane)) = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) bytes[value_at(r, 4 * lane + e)] = (uint8_t)q[e];
        }
    };
#pragma unroll
    for (int i = 0; i < KEEP; i++)
        if (lo + i < hi) write(kept[i], lo + i);
    for (int r = lo + KEEP; r < hi; r++) {
        float v[4];
        load(v, r);
        write(v, r);
    }
    __syncwarp();  // (every lane has the old header)
    if (lane == 0) *((uint2*)unit + kind) = make_uint2(__float_as_uint(scale), bad);
}

// A few rows a sequence (a decoding step): a warp for each (sequence, block, KV head, keys or values).
template <int HD, typename T>
__global__ void __launch_bounds__(128) append_few_kernel(Kv8Cache c, Kv8Seqs sq, Kv8Rows x, uint32_t tiles, uint32_t units, int keep_behind, int aligned, uint32_t* status) {
    pdl_launch_dependents();
    const uint32_t at = blockIdx.x * 4 + (threadIdx.x >> 5), kind = at & 1, head = (at >> 1) % c.nkv, rest = (at >> 1) / c.nkv, tile = rest % tiles, s = rest / tiles;
    pdl_wait();
    Seq seq;
    if (at >= units || !sequence(sq, s, &seq, status) || seq.count == 0) return;
    const uint32_t end = seq.start + seq.count, b_end = (end - 1) / KV8_BLOCK + 1;
    const T* const from = (const T*)(kind ? x.v : x.k) + (size_t)head * x.hs;
    for (uint32_t b = seq.start / KV8_BLOCK + tile; b < b_end; b += tiles) {
        const int base = (int)(b * KV8_BLOCK), lo = max((int)seq.start - base, 0), hi = min((int)end - base, (int)KV8_BLOCK);
        const uint32_t staying = rows_staying(lo, hi, keep_behind);
        const int id = block_of(c, sq, s, b, status);
        if (id < 0) continue;
        uint8_t* const unit = c.units + ((size_t)id * c.nkv + head) * unit_bytes(HD);
        append_rows<HD, T>(unit, kind, staying ? *((const uint2*)unit + kind) : make_uint2(0, 0), lo, hi, staying,
                           from + (size_t)(seq.r0 + (uint32_t)(base + lo) - seq.start) * x.rs, x.rs, aligned);
    }
}

// A decoding step's token: its queries rotated, its keys and values into the cache; a CTA a head, a thread a dimension (rope_head).
template <int HD>
__global__ void __launch_bounds__(HD) rope_append_kernel(Kv8Cache c, const float* __restrict__ qkv, float* __restrict__ qo, const float* __restrict__ qn,
                                                         const float* __restrict__ kn, const float* __restrict__ cs_table, const uint32_t* __restrict__ sp, DecRope p) {
    __shared__ __align__(16) float row[HD];
    __shared__ float buf[256], red[32];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t h = blockIdx.x, pos = sp[0];
    const bool is_query = h < p.nh;
    const uint32_t kind = h >= p.nh + p.nkv, head = is_query ? 0 : h - p.nh - kind * p.nkv, b = pos / KV8_BLOCK;
    if (!is_query && b >= c.n_blocks) return;  // (the host refuses the step before this)
    uint8_t* const unit = c.units + ((size_t)b * c.nkv + head) * unit_bytes(HD);
    const int lo = (int)(pos % KV8_BLOCK);
    const uint32_t staying = rows_staying(lo, lo + 1, 0);
    uint2 old = make_uint2(0, 0);
    if (!is_query && staying && threadIdx.x < 32) old = *((const uint2*)unit + kind);
    p.max_len = 1;  // (heads one behind the other: this one's row)
    attend_core::rope_head<float>(h, threadIdx.x, pos, sp[1], 0, qkv, qo, row - (size_t)head * HD, row - (size_t)head * HD, qn, kn, cs_table, p, buf, red);
    if (!is_query && threadIdx.x < 32) append_rows<HD, float>(unit, kind, old, lo, lo + 1, staying, row, HD, true);
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

// The same of a few rows a sequence: a warp for each (sequence, block, KV head, keys or values), and no more of a unit than they have.
template <int HD>
__global__ void __launch_bounds__(128) read_few_kernel(Kv8Cache c, Kv8Seqs sq, float* __restrict__ k, float* __restrict__ v, uint32_t tiles, uint32_t units, uint32_t* status) {
    constexpr int UNIT = (int)unit_bytes(HD), LANES = HD / 4;
    const int lane = threadIdx.x & 31, d = 4 * (lane % LANES);
    const uint32_t at = blockIdx.x * 4 + (threadIdx.x >> 5), kind = at & 1, head = (at >> 1) % c.nkv, rest = (at >> 1) / c.nkv, tile = rest % tiles, s = rest / tiles;
    Seq seq;
    if (at >= units || !sequence(sq, s, &seq, status) || seq.count == 0) return;
    const uint32_t end = seq.start + seq.count, b_end = (end - 1) / KV8_BLOCK + 1;
    for (uint32_t b = seq.start / KV8_BLOCK + tile; b < b_end; b += tiles) {
        const int id = block_of(c, sq, s, b, status);
        if (id < 0) continue;
        const uint8_t* const unit = c.units + ((size_t)id * c.nkv + head) * UNIT;
        const uint2 header = *((const uint2*)unit + kind);
        const uint8_t* const bytes = unit + KV8_HEADER + kind * (KV8_BLOCK * HD);
        const int base = (int)(b * KV8_BLOCK), lo = max((int)seq.start - base, 0), hi = min((int)end - base, (int)KV8_BLOCK);
        for (int r = lo + lane / LANES; r < hi; r += 32 / LANES) {
            const float scale = (header.y >> r) & 1 ? NAN : __uint_as_float(header.x);
            uchar4 q;
            if (kind == 0) q = *(const uchar4*)(bytes + key_at<HD>(r, d));
            else q = make_uchar4(bytes[value_at(r, d)], bytes[value_at(r, d + 1)], bytes[value_at(r, d + 2)], bytes[value_at(r, d + 3)]);
            const auto value = [&](unsigned char x) { return (float)((int)x - 128) * scale; };
            *(float4*)((kind ? v : k) + ((size_t)(seq.r0 + (uint32_t)(base + r) - seq.start) * c.nkv + head) * HD + d) = make_float4(value(q.x), value(q.y), value(q.z), value(q.w));
        }
    }
}

// Blocks that the rows of one sequence may reach into.
uint32_t tiles_of(const Kv8Seqs& s) { return (uint32_t)(((size_t)s.max_rows + 2 * KV8_BLOCK - 2) / KV8_BLOCK); }

template <int HD, typename T>
cudaError_t append_t(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Rows& x, bool keep_behind, uint32_t* status, cudaStream_t st, bool pdl) {
    uint32_t tiles = tiles_of(s);
    const size_t most = 0x7fffffffu / ((size_t)c.nkv * s.n_seqs * 2);
    if (most == 0) return cudaErrorInvalidValue;
    if (tiles > most) tiles = (uint32_t)most;
    const size_t unit = 4 * sizeof(T);
    const size_t places = (uintptr_t)x.k | (uintptr_t)x.v | x.rs * sizeof(T) | x.hs * sizeof(T);
    const int aligned = (places & (unit - 1)) == 0, wide = (places & 15) == 0;
    // 8 KV heads of 128, us, a warp / a CTA a block: a sequence's one row 2.3 / 3.2, four 3.0 / 3.3; 64 sequences 2.8 / 5.4, 5.3 / 6.3; 256 sequences of one row 5.4 / 14.3, four
    // 9.5 / 14.2, six 13.2 / 14.4, eight 16.8 / 14.3.
    if (s.max_rows <= FEW) {
        const uint32_t units = 2 * tiles * c.nkv * s.n_seqs;
        return launch_k(append_few_kernel<HD, T>, dim3((units + 3) / 4), dim3(128), 0, st, pdl, c, s, x, tiles, units, keep_behind ? 1 : 0, aligned, status);
    }
    tiles = std::min<uint32_t>(tiles, std::max<uint32_t>(1, (uint32_t)(KV_WAVE * 148 / ((size_t)c.nkv * s.n_seqs))));
    return launch_k(append_kernel<HD, T>, dim3(tiles * c.nkv * s.n_seqs), dim3(KV_THREADS), 0, st, pdl, c, s, x, tiles, keep_behind ? 1 : 0, wide, status);
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

cudaError_t launch_rope_kv8(const Kv8Cache& c, const float* qkv, float* qo, const float* qn, const float* kn, const float* cs_table, const uint32_t* sp, const DecRope& p,
                            cudaStream_t st, bool pdl) {
    if (!kv8_supports(c.nkv, c.hd) || p.hd != c.hd || p.nkv != c.nkv) return cudaErrorInvalidValue;
    const dim3 grid(p.nh + 2 * p.nkv);
    return c.hd == 64 ? launch_k(rope_append_kernel<64>, grid, dim3(64), 0, st, pdl, c, qkv, qo, qn, kn, cs_table, sp, p)
                      : launch_k(rope_append_kernel<128>, grid, dim3(128), 0, st, pdl, c, qkv, qo, qn, kn, cs_table, sp, p);
}

cudaError_t launch_kv8_read(const Kv8Cache& c, const Kv8Seqs& s, float* k, float* v, uint32_t* status, cudaStream_t st) {
    if (!kv8_supports(c.nkv, c.hd)) return cudaErrorInvalidValue;
    if (s.n_seqs == 0 || s.n_rows == 0 || s.max_rows == 0) return cudaSuccess;
    uint32_t tiles = tiles_of(s);
    const size_t most = 0x7fffffffu / ((size_t)c.nkv * s.n_seqs * 2);
    if (most == 0) return cudaErrorInvalidValue;
    if (tiles > most) tiles = (uint32_t)most;
    // 64 sequences, 8 KV heads of 128, us, a warp / a CTA a block: one row 2.1 / 3.1, four 3.6 / 4.0, eight 5.4 / 4.2.
    if (s.max_rows <= FEW) {
        const uint32_t units = 2 * tiles * c.nkv * s.n_seqs;
        if (c.hd == 64) read_few_kernel<64><<<(units + 3) / 4, 128, 0, st>>>(c, s, k, v, tiles, units, status);
        else read_few_kernel<128><<<(units + 3) / 4, 128, 0, st>>>(c, s, k, v, tiles, units, status);
        return cudaGetLastError();
    }
    if (c.hd == 64) read_kernel<64><<<tiles * c.nkv * s.n_seqs, KV_THREADS, 0, st>>>(c, s, k, v, tiles, status);
    else read_kernel<128><<<tiles * c.nkv * s.n_seqs, KV_THREADS, 0, st>>>(c, s, k, v, tiles, status);
    return cudaGetLastError();
}

}  // namespace b2
