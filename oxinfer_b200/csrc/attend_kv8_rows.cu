// Attention over the 8-bit cache for many rows of a sequence on tcgen05: S = Q K^T and O += P V with f16 operands and f32 sums in tensor memory, softmax by two
// threads a row (attend_rows.cu has the form for f16 caches). The integers are exact as f16; a block's scale of keys multiplies its 32 columns of scores, a
// block's scale of values, over the largest that the CTA's rows see, goes into the f16 values (a power of two, exact down to 2^-29 of the largest). Where values lie
// further apart, the CTA's sums of values are made anew without tensor cores (far_sums): a row may see the small ones only.
// Queries are rounded to f16 after a power of two that brings each row's largest to 1 .. 2, probabilities to f16.
//
// A CTA takes 256 rows of a KV head (query heads token by token, two tiles of 128) and key tiles of 128, four blocks:
//   warps 0..15  : softmax, two warps a row, a thread each: 0..3 and 4..7 have the first and the third block of the two tiles' rows, 8..15 the others; and the rows out;
//   warps 16, 17 : issue a tile's instructions;
//   warp 18      : copies the blocks' units as they lie in the cache (bulk copies), a place for each block of a tile;
//   warps 20..23 : expand them, a warp a block: bytes to f16, into swizzled tiles, keys as rows, values as rows of a dimension with the keys along them. Key r of a block in
//                  both is token 16 (r / 4 % 2) + 4 (r / 8) + r % 4: eight keys of a dimension are eight bytes of a lane's word, one store of 16 bytes.
// Expanded tiles are two slots deep, so the next tile is expanded under the current one's products. A warp's reads and its stores of 16 bytes meet no bank
// twice. Probabilities take the place of the first half of a tile's scores; the next tile's second half is multiplied, and taken in, while they are still at work. Few rows over
// many keys: Z CTAs of a cluster take a share of the key tiles each, and add their sums through shared memory.
//
// What bounds it: a softmax warp's chain for a tile of keys, 3700 cycles without a cap (scores out of tensor memory and their largest 830, the row's two warps' meeting and the turn 870,
// exponentials 1330 of which the exponential unit needs 1024, the rest waits for products), 5600 with one. The row tiles take turns at the exponentials: left to themselves they
// meet there, and the tensor cores, 2048 cycles of 3700, idle while both wait for products (136 us instead of 110, turns handed on at half of them 119). 2048 tokens of 32 heads over 8 KV heads
// of 128 behind 2048 more (103 GFLOP): 112 us, 920 TFLOP/s; with a cap 170 us (replays). On mma.sync (attend_kv8.cu) 741 and 940. Steps, without / with a cap: bytes expanded by four
// warps a block and everyone in step 164 us, a warp a block 142, descriptors in the warp's registers and places by turned bits 132, turns 115, a shorter start 106 / 187, two
// warps a row 120 / 181, each with a block of both halves of the keys 110 / 170. Short prompts (five of 185 to 542 tokens with 12 heads 25.3 us, half of it in the
// tiles) pay for the CTA's start: the largest scale of values is looked for by the warps that expand, while the others take in the queries, eight values a lane (33 us before; one warp
// a row 27.8). No gain: what goes into the exponentials made ahead of a tile's turn, their sums behind it; the two warps of a row at a barrier of the hardware's (110 -> 109.4).
#include <cfloat>
#include <type_traits>

#include "gemm_wt.h"
#include "kv8.cuh"
#include "pdl.cuh"
#include "tcgen05.cuh"

namespace b2 {

using namespace kv8;

namespace {

constexpr int KT_THREADS = 768, KT_TILE = 128, KT_BLOCKS = KT_TILE / (int)KV8_BLOCK;
constexpr uint32_t KT_TMEM_COLS = 512;
// tanh(z) / z by powers of z^2
constexpr float K0 = 0.999999464f, K1 = -0.333283484f, K2 = 0.132598311f, K3 = -0.0500801913f, K4 = 0.0129507277f;
constexpr float LAZY_BITS = 8.0f;  // the sums are brought to a new largest score only where it is 2^8 times the one they are at
constexpr float KT_P_BITS = 7.0f;  // probabilities are held 2^7 times as large, up to 2^15: those below 2^-21 of the largest lose bits, below 2^-32 they are zeros (at 2^0 a long flat tail got lost)
// The sums leave tensor memory 2^32 times as small, so that they stay finite where the values are (KT_P_BITS + LAZY_BITS, and up to 2^17 keys of a row).
constexpr float KT_SUM_DOWN = 0x1p-32f, KT_SUM_UP = 0x1p32f;
constexpr float V_ONE = 32.0f;  // the largest scale of values as it enters the f16 values: 1152 of it has to be an f16, too

struct __align__(16) KtShared {
    float told[2][2 * KT_TILE];             // what the two warps of a row tell one another, a half of the keys each; in the beginning [0] is what the rows' scores are multiplied by
    // of a tile's blocks, four tiles in turn: a tile's are written once the scores of two tiles ahead have been made, so the softmax of three tiles ahead is done
    float k_scale[4][KT_BLOCKS];
    uint32_t bad[4][KT_BLOCKS];             // tokens that count as NaN
    uint64_t k_full[2], v_full[2], k_empty[2], v_empty[2], q_full, s_full[2][2], s_free[2], p_full[2][2], o_full, u_full[KT_BLOCKS], u_empty[KT_BLOCKS], turn[2], pair[2][4];
    uint32_t tmem_base, v_top, item_seq, item_block;
    volatile uint32_t far;                  // a block's values are below what f16 holds beside the largest
    struct {
        Seq seq;
        uint32_t prefix, b_beg, b_end, r_block, r_end;
    } place;                                // (far_sums: nobody else keeps them in registers for it)
    volatile uint32_t abort_flag;
};

template <int HD>
struct KtSizes {
    static constexpr uint32_t TILE = KT_TILE * HD * 2, UNIT = unit_bytes(HD);
    static constexpr uint32_t Q = 0, K = 2 * TILE, V = 4 * TILE, RING = 6 * TILE;
    static constexpr uint32_t SHARED = RING + KT_BLOCKS * UNIT;
    static constexpr size_t NEED = SHARED + sizeof(KtShared);
    static constexpr size_t BYTES = NEED < TMEM_512_SMEM ? TMEM_512_SMEM : NEED;  // (one CTA an SM: it takes all of the tensor memory)
    static_assert(BYTES <= 227 * 1024 && SHARED % alignof(KtShared) == 0);
};

struct KtArgs {
    Kv8Cache c;
    Kv8Seqs sq;
    const void* q;
    void* out;
    size_t q_stride, out_stride;
    uint32_t G, g_inv, window, blocks;  // g_inv: ceil(2^32 / G), 0 for one head; blocks: of 256 rows, all sequences', as far as the grid goes
    float c2, q_sign, cap2, cap_z;      // |scale| in powers of two and its sign; cap in powers of two, and what brings scores in powers of two to score / cap
    const float* slopes;
    const int32_t* prefix;
    int aligned, wide;                  // queries and results: four values to their size, eight 16-bit ones to 16 bytes
    uint32_t Z;
    uint32_t* status;
};

// Bounded as mbar_wait is: false when the CTA gives up.
__device__ __forceinline__ bool kt_wait(uint64_t* bar, uint32_t parity, KtShared* sh, uint32_t* status, bool heed_abort = true) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    for (uint32_t spin = 1;; spin++) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((spin & 255) == 0) {
            if (heed_abort && sh->abort_flag) return false;
            if (clock64() - t0 > WAIT_LIMIT_CYCLES) {
                *(volatile uint32_t*)status = KV8_TIMEOUT;
                sh->abort_flag = 1;
                return false;
            }
        }
    }
}
__device__ __forceinline__ void kt_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void kt_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
        "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
          "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]),
          "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void kt_ld8(uint32_t taddr, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void kt_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void kt_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void kt_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void kt_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void kt_mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ float kt_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t kt_pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *(const uint32_t*)&h;
}
// Four bytes q + 128 as f16 values q times s: 1024 + byte by its bits, s and -1152 s.
__device__ __forceinline__ uint2 kt_expand(uint32_t w, __half2 s, __half2 b) {
    const uint32_t x = __byte_perm(w, 0x64646464u, 0x4140u), y = __byte_perm(w, 0x64646464u, 0x4342u);
    const __half2 u = __hfma2(*(const __half2*)&x, s, b), v = __hfma2(*(const __half2*)&y, s, b);
    return make_uint2(*(const uint32_t*)&u, *(const uint32_t*)&v);
}
__device__ __forceinline__ void kt_sts(uint32_t at, uint2 a, uint2 b) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a.x), "r"(a.y), "r"(b.x), "r"(b.y) : "memory");
}
__device__ __forceinline__ uint32_t kt_token(const KtArgs& a, uint32_t r) { return a.g_inv ? __umulhi(r, a.g_inv) : r; }
// The token (of a block's 32) that key r of an expanded block is.
__device__ __forceinline__ constexpr uint32_t kt_tok(uint32_t r) { return 16 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3); }
template <typename T>
__device__ __forceinline__ void kt_store4(T* p, float4 v, bool aligned) {
    if constexpr (sizeof(T) == 4) {
        if (aligned) *(float4*)p = v;
        else p[0] = v.x, p[1] = v.y, p[2] = v.z, p[3] = v.w;
    } else {
        alignas(8) T t[4];
        const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (std::is_same<T, __half>::value) t[i] = __float2half_rn(f[i]);
            else t[i] = __float2bfloat16_rn(f[i]);
        }
        if (aligned) *(uint2*)p = *(const uint2*)t;
        else {
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = t[i];
        }
    }
}

__device__ __forceinline__ float4 kt_peer_f4(const void* p, uint32_t cta) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr(p, cta)) : "memory");
    return v;
}
__device__ __forceinline__ float2 kt_peer_f2(const void* p, uint32_t cta) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_addr(p, cta)) : "memory");
    return v;
}

// The sums of sixteen rows from `at0` of the CTA's on, over the CTA's share of the keys, without tensor cores: values go into f32 sums with their blocks' own scales. A warp has a row at a
// time, a lane a key of a block for the scores, then HD / 32 dimensions of the values. m: lane i & 15's is the largest score of row i as far as it was kept. qs: [HD] of the warp's own.
// Some 16 instructions a key and row: 2048 tokens of 32 heads behind 2048 take 9.7 ms instead of 0.11. Values 2^29 apart are hardly ever met; looking for them costs others 0.3 to 1 %.
template <int HD, bool SPECIAL, typename T>
__device__ __forceinline__ void far_sums(const KtArgs& a, const KtShared* sh, uint32_t at0, float m, float* qs, uint8_t* sums, float2* ml) {
    constexpr int D = HD / 32;
    const int lane = threadIdx.x & 31;
    const uint32_t s = sh->item_seq, head = blockIdx.x / a.Z % a.c.nkv;
    const Seq seq = sh->place.seq;
    const uint32_t prefix = sh->place.prefix, b_beg = sh->place.b_beg, b_end = sh->place.b_end, r_block = sh->place.r_block, r_end = sh->place.r_end;
#pragma unroll 1
    for (uint32_t at = at0; at < at0 + 16 && r_block + at < r_end; at++) {
        const uint32_t r = r_block + at, tok = kt_token(a, r), h = head * a.G + (r - tok * a.G), qp = seq.start + tok;
        const T* const q = (const T*)a.q + (size_t)(seq.r0 + tok) * a.q_stride + (size_t)h * HD;
        float x[D];
        uint32_t bits = 0;
#pragma unroll
        for (int k = 0; k < D; k++) {
            x[k] = to_f32<T>(q[lane + 32 * k]);
            bits = max(bits, __float_as_uint(x[k]) & 0x7fffffffu);
        }
        bits = __reduce_max_sync(0xffffffffu, bits);
        const int ex = min(max((int)(bits >> 23), 40), 254) - 127;
        const float down = (ex == 127 ? 0x1p-127f : pow2(-ex)) * a.q_sign, qf = (bits >= 0x7f800000u ? NAN : pow2(ex)) * a.c2;
#pragma unroll
        for (int k = 0; k < D; k++) qs[lane + 32 * k] = x[k] * down;
        __syncwarp();
        const float top = __shfl_sync(0xffffffffu, m, at & 15), base = top == -INFINITY ? 0.0f : KT_P_BITS - top;
        const float slope = SPECIAL && a.slopes ? a.slopes[h] * 1.44269504f : 0.0f;
        const uint32_t see_to = max(qp + 1, prefix), see_from = a.window != 0 && qp + 1 > a.window ? qp + 1 - a.window : 0u;
        const uint32_t b1 = min(b_end, (see_to + KV8_BLOCK - 1) / KV8_BLOCK);
        float o[D] = {}, den = 0.0f;
#pragma unroll 1
        for (uint32_t b = max(b_beg, see_from / KV8_BLOCK); b < b1; b++) {
            const int id = max(block_of(a.c, a.sq, s, b, a.status), 0);
            const uint8_t* const unit = a.c.units + ((size_t)id * a.c.nkv + head) * unit_bytes(HD);
            const Header hd = *(const Header*)unit;
            float dot = 0.0f;
#pragma unroll 1
            for (int d = 0; d < HD; d += 16) {
                const uint4 w4 = *(const uint4*)(unit + KV8_HEADER + key_at<HD>(lane, d));
                const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                for (int e = 0; e < 16; e++) dot = fmaf(qs[d + e], (float)((int)((w[e >> 2] >> (8 * (e & 3))) & 0xffu) - 128), dot);
            }
            const uint32_t j = b * KV8_BLOCK + lane;
            float y = dot * (qf * hd.k_scale);
            if (SPECIAL && a.cap2 > 0.0f) y = a.cap2 * tanhf(y * a.cap_z);
            if (SPECIAL && a.slopes) y = fmaf(slope, (float)((int)j - (int)qp), y);
            if (((hd.k_bad | hd.v_bad) >> lane) & 1) y = NAN;
            const float p = j >= see_from && j < see_to ? kt_exp2(y + base) : 0.0f, scale = hd.v_scale * KT_SUM_DOWN;
            den += p;
            float part[D] = {};
#pragma unroll 1
            for (int t = 0; t < 4; t++) {  // tokens 4 t .. and 16 + 4 t ..
                uint2 w[D];
#pragma unroll
                for (int k = 0; k < D; k++) w[k] = *(const uint2*)(unit + KV8_HEADER + KV8_BLOCK * HD + value_at(4 * t, lane + 32 * k));
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float pe = __shfl_sync(0xffffffffu, p, 16 * (e >> 2) + 4 * t + (e & 3));
#pragma unroll
                    for (int k = 0; k < D; k++) part[k] = fmaf(pe, (float)((int)(((e < 4 ? w[k].x : w[k].y) >> (8 * (e & 3))) & 0xffu) - 128), part[k]);
                }
            }
#pragma unroll
            for (int k = 0; k < D; k++) o[k] = fmaf(part[k], scale, o[k]);
        }
#pragma unroll
        for (int i = 16; i > 0; i >>= 1) den += __shfl_xor_sync(0xffffffffu, den, i);
#pragma unroll
        for (int k = 0; k < D; k++) {
            const uint32_t d = lane + 32 * k;
            ((float*)(sums + (size_t)at * HD * 4))[4 * ((d >> 2) ^ (at & 7)) + (d & 3)] = o[k];
        }
        if (lane == 0) ml[at] = make_float2(top, a.Z > 1 ? den : den > 0.0f || den != den ? KT_SUM_UP / den : 0.0f);
        __syncwarp();  // (the row's queries have been read)
    }
}

// Grid: (block of 256 rows, KV head, share of the keys), shares first (a cluster's Z), then heads; the blocks of all sequences one after another, a sequence's last
// first. SPECIAL: a cap or a bias.
template <int HD, bool SPECIAL, typename T>
__global__ void __launch_bounds__(KT_THREADS, 1) attend_kv8_rows_kernel(const __grid_constant__ KtArgs a) {
    using L = KtSizes<HD>;
    constexpr uint32_t HALF = KT_TILE * 128, VHALF = HD * 128;  // 64 dimensions of all keys; 64 keys of all dimensions
    extern __shared__ __align__(1024) uint8_t smem[];  // (the kernel has no other shared memory: tiles begin on the 1024 bytes that their swizzle needs)
    KtShared* const sh = (KtShared*)(smem + L::SHARED);
    // (what the instructions' descriptors are made of is known to be the warp's: registers of the warp, no moves into them ahead of every instruction)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t z = blockIdx.x % a.Z, unit_no = blockIdx.x / a.Z, head = unit_no % a.c.nkv, want = unit_no / a.c.nkv;
    pdl_launch_dependents();
    pdl_wait();
    // ---------------- which sequence, and which of its blocks of rows ----------------
    if (warp == 0) {
        uint32_t before = 0, found = 0xffffffffu, blk = 0;
        for (uint32_t s0 = 0; s0 < a.sq.n_seqs && found == 0xffffffffu; s0 += 32) {
            const uint32_t s = s0 + lane;
            Seq q;
            const uint32_t nb = s < a.sq.n_seqs && sequence(a.sq, s, &q, a.status) ? (uint32_t)(((size_t)q.count * a.G + 2 * KT_TILE - 1) / (2 * KT_TILE)) : 0u;
            uint32_t upto = nb;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, nb > 0 && want >= before + upto - nb && want < before + upto);
            if (hit) {
                const int at = __ffs(hit) - 1;
                found = s0 + at;
                const uint32_t end = __shfl_sync(0xffffffffu, before + upto, at);
                blk = end - 1 - want;  // (the last block, with the most keys, first)
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) {
            sh->item_seq = found;
            sh->item_block = blk;
            sh->v_top = 0;
            sh->far = 0;
            sh->abort_flag = 0;
        }
    }
    __syncthreads();
    const uint32_t s = sh->item_seq;
    if (s == 0xffffffffu) return;
    Seq seq;
    if (!sequence(a.sq, s, &seq, a.status)) return;
    const uint32_t rows = seq.count * a.G, len = seq.start + seq.count, r_block = sh->item_block * (2 * KT_TILE), r_end = min(r_block + 2 * KT_TILE, rows);
    const uint32_t prefix = a.prefix ? (uint32_t)min(max(a.prefix[s], 0), (int)len) : 0;
    const int tiles = r_block + KT_TILE < r_end ? 2 : 1;
    const uint32_t first_qp = seq.start + kt_token(a, r_block), last_qp = seq.start + kt_token(a, r_end - 1);
    auto first_key = [&](uint32_t qp) { return a.window != 0 && qp + 1 > a.window ? qp + 1 - a.window : 0u; };
    const uint32_t all_beg = first_key(first_qp) / KV8_BLOCK, all_end = (max(last_qp + 1, prefix) + KV8_BLOCK - 1) / KV8_BLOCK;
    const uint32_t all_0 = all_beg / KT_BLOCKS, all_n = (all_end + KT_BLOCKS - 1) / KT_BLOCKS - all_0, share = (all_n + a.Z - 1) / a.Z;  // tiles of 128 keys
    const int n = (int)(z * share < all_n ? min(share, all_n - z * share) : 0u);                                                          // this CTA's
    const uint32_t b_0 = (all_0 + z * share) * KT_BLOCKS, b_beg = max(all_beg, b_0), b_end = max(b_beg, min(all_end, b_0 + n * KT_BLOCKS));

    if (tid == 0) {
        sh->place = {seq, prefix, b_beg, b_end, r_block, r_end};
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh->k_full[i], 4);
            mbar_init(&sh->v_full[i], 4);
            mbar_init(&sh->k_empty[i], tiles);
            mbar_init(&sh->v_empty[i], tiles);
            mbar_init(&sh->s_full[i][0], 1);
            mbar_init(&sh->s_full[i][1], 1);
            mbar_init(&sh->s_free[i], 8);
            mbar_init(&sh->p_full[i][0], 8);
            mbar_init(&sh->p_full[i][1], 8);
            for (int q = 0; q < 4; q++) mbar_init(&sh->pair[i][q], 2);
        }
        for (int i = 0; i < KT_BLOCKS; i++) {
            mbar_init(&sh->u_full[i], 1);
            mbar_init(&sh->u_empty[i], 1);
        }
        mbar_init(&sh->q_full, 16);
        mbar_init(&sh->o_full, 2);
        mbar_init(&sh->turn[0], 8);
        mbar_init(&sh->turn[1], 8);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem_base)), "r"(KT_TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh->tmem_base, 0);

    // 768 threads are launched with 80 registers each: 512 x 96 + 128 x 40 + 128 x 56 of them.
    if (warp >= 20) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;" ::: "memory");
        // ---------------- bytes to f16: a warp for each block of a tile ----------------
        const uint32_t bq = warp - 20, t = lane & 3, n0 = (lane >> 2) & 1, u2 = lane >> 3;
        const __half2 one = __float2half2_rn(1.0f), off = __float2half2_rn(-1152.0f);
        float low = INFINITY;
        {  // the largest scale of values that the rows may see
            uint32_t top = 0;
#pragma unroll 4
            for (uint32_t b = b_beg + tid - 640; b < b_end; b += 128) {
                const int id = block_of(a.c, a.sq, s, b, a.status);
                const float v = ((const Header*)(a.c.units + ((size_t)max(id, 0) * a.c.nkv + head) * L::UNIT))->v_scale;
                top = max(top, __float_as_uint(fmaxf(v, 0.0f)));
                low = v > 0.0f ? fminf(low, v) : low;
            }
            top = __reduce_max_sync(0xffffffffu, top);
            if (lane == 0 && top) atomicMax(&sh->v_top, top);
            asm volatile("bar.sync 2, 128;" ::: "memory");
        }
        const float v_top = __uint_as_float(*(volatile uint32_t*)&sh->v_top);
        const float v_inv = v_top > 0.0f ? V_ONE / v_top : 0.0f;
        if (__any_sync(0xffffffffu, low * v_inv < 0x1p-24f)) {  // (seldom: f16 values would be zero; a block of zeros has the smallest scale, so the warp looks at its bytes)
            bool found = false;
#pragma unroll 1
            for (uint32_t b0 = b_beg + (warp - 20) * 32; b0 < b_end && !found; b0 += 128) {
                const int id = b0 + lane < b_end ? max(block_of(a.c, a.sq, s, b0 + lane, a.status), 0) : 0;
                const unsigned long long at = (unsigned long long)(a.c.units + ((size_t)id * a.c.nkv + head) * L::UNIT);
                const float v = b0 + lane < b_end ? ((const Header*)at)->v_scale : 0.0f;
#pragma unroll 1
                for (uint32_t left = __ballot_sync(0xffffffffu, v > 0.0f && v * v_inv < 0x1p-24f); left && !found; left &= left - 1) {
                    const uint4* const bytes = (const uint4*)(__shfl_sync(0xffffffffu, at, __ffs(left) - 1) + KV8_HEADER + KV8_BLOCK * HD);
                    uint32_t any = 0;
#pragma unroll
                    for (uint32_t k = 0; k < KV8_BLOCK * HD / 512; k++) {
                        const uint4 w = bytes[32 * k + lane];
                        any |= (w.x ^ 0x80808080u) | (w.y ^ 0x80808080u) | (w.z ^ 0x80808080u) | (w.w ^ 0x80808080u);
                    }
                    found = __any_sync(0xffffffffu, any != 0);
                }
            }
            if (found && lane == 0) sh->far = 1;
            __syncwarp();
        }
        const uint8_t* const unit = smem + L::RING + bq * L::UNIT;
        const int skipped = b_0 + bq < b_beg ? 1 : 0;
        for (int i = 0; i < n; i++) {
            const int slot = i & 1;
            const uint32_t b = b_0 + i * KT_BLOCKS + bq, back = (uint32_t)(((i >> 1) - 1) & 1);
            const bool there = b >= b_beg && b < b_end;
            if (there && !__all_sync(0xffffffffu, kt_wait(&sh->u_full[bq], (uint32_t)((i - skipped) & 1), sh, a.status))) break;
            if (i >= 2 && !__all_sync(0xffffffffu, kt_wait(&sh->k_empty[slot], back, sh, a.status))) break;
            const Header h = *(const Header*)unit;
            if (lane == 0) {
                sh->k_scale[i & 3][bq] = there ? h.k_scale : 0.0f;
                sh->bad[i & 3][bq] = there ? h.k_bad | h.v_bad : 0u;
            }
            // Keys: lanes (t, n % 2) read eight banks, and their rows' places in the swizzle differ: of a head of 128 the upper half of the lanes takes the other
            // tile of two. A place is the lane's own with bits of the step's turned.
            uint8_t* const kd = smem + L::K + slot * L::TILE;
            if (there) {
                const uint32_t nn = n0 + 2 * u2, t1 = t >> 1, c0 = HD == 128 ? ((t & 1) * 4) ^ (2 * t1) : t * 2, r0 = HD == 128 ? 2 * t1 + n0 : n0;
                const uint8_t* const from = unit + KV8_HEADER + (nn * 4 + t) * 16;
                const uint8_t* const from_tile[2] = {from + (HD == 128 ? t1 * 1024 : 0u), from - (HD == 128 ? t1 * 1024 : 0u)};
                const uint32_t to = smem_u32(kd) + (HD == 128 ? t1 * HALF : 0u) + (KV8_BLOCK * bq + 8 * (nn >> 1) + r0) * 128 + ((c0 ^ n0) << 4);
#pragma unroll
                for (uint32_t k = 0; k < 4 * HD / 64; k++) {
                    const uint32_t hf = HD == 128 ? k & 1 : 0, jb = HD == 128 ? k >> 1 : k;
                    const uint4 w = *(const uint4*)(from_tile[jb & 1] + jb * (8 * HD) + hf * 512);
                    const uint2 x0 = kt_expand(w.x, one, off), x1 = kt_expand(w.y, one, off), x2 = kt_expand(w.z, one, off), x3 = kt_expand(w.w, one, off);
                    const uint32_t at = to ^ ((2 * jb) << 7) ^ ((2 * jb ^ 2 * hf) << 4);
                    kt_sts(at, x0, x1);
                    kt_sts(at ^ 16, x2, x3);
                }
            } else {
                for (uint32_t x = lane; x < KV8_BLOCK * 8 * (HD / 64); x += 32)
                    *(uint4*)(kd + (x / (KV8_BLOCK * 8)) * HALF + KV8_BLOCK * bq * 128 + x % (KV8_BLOCK * 8) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->k_full[slot]);
            if (i >= 2 && !__all_sync(0xffffffffu, kt_wait(&sh->v_empty[slot], back, sh, a.status))) break;
            const float vs = there ? h.v_scale * v_inv : 0.0f;
            const __half2 v_s = __float2half2_rn(vs), v_b = __hmul2(v_s, off);  // (exact; both zero where the scale is below an f16's smallest)
            // values: 16 dimensions at a time
            uint8_t* const vd = smem + L::V + slot * L::TILE + (bq >> 1) * VHALF;
            const uint32_t g = n0 + 2 * (u2 & 1) + 4 * ((u2 >> 1) ^ n0), cc = (bq & 1) * 4 + t;
            const uint32_t to = smem_u32(vd) + g * 128 + ((cc ^ g) << 4);  // (dimensions d and d + 8 have one place in the swizzle)
            if (there) {
                const uint8_t* const from = unit + KV8_HEADER + KV8_BLOCK * HD + (g * 4 + t) * 16;
#pragma unroll
                for (uint32_t gi = 0; gi < HD / 16; gi++) {
                    const uint4 w = *(const uint4*)(from + gi * 512);
                    const uint2 x0 = kt_expand(w.x, v_s, v_b), x1 = kt_expand(w.y, v_s, v_b), x2 = kt_expand(w.z, v_s, v_b), x3 = kt_expand(w.w, v_s, v_b);
                    kt_sts(to + gi * 2048, x0, x1);
                    kt_sts(to + gi * 2048 + 1024, x2, x3);
                }
            } else {
#pragma unroll
                for (uint32_t gi = 0; gi < HD / 16; gi++) {
                    kt_sts(to + gi * 2048, make_uint2(0, 0), make_uint2(0, 0));
                    kt_sts(to + gi * 2048 + 1024, make_uint2(0, 0), make_uint2(0, 0));
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh->v_full[slot]);
                if (there) mbar_arrive(&sh->u_empty[bq]);
            }
        }
    } else if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;" ::: "memory");
        if (warp == 18) {
            // ---------------- units: block q of a tile into place q ----------------
            int ids = 0;
            bool ok = true;
            uint32_t b = b_beg;
            for (; b < b_end; b++) {
                const uint32_t at = b - b_0, q = at % KT_BLOCKS, before = at / KT_BLOCKS - (b_0 + q < b_beg ? 1 : 0);  // units that this place has had
                if (((b - b_beg) & 31) == 0) ids = b + lane < b_end ? max(block_of(a.c, a.sq, s, b + lane, a.status), 0) : 0;
                const int id = __shfl_sync(0xffffffffu, ids, (b - b_beg) & 31);
                if (before > 0) ok = __all_sync(0xffffffffu, kt_wait(&sh->u_empty[q], (before - 1) & 1, sh, a.status));
                if (!ok) break;
                if (elect_one()) {
                    mbar_arrive_expect_tx(&sh->u_full[q], L::UNIT);
                    kt_bulk(smem + L::RING + q * L::UNIT, a.c.units + ((size_t)id * a.c.nkv + head) * L::UNIT, L::UNIT, &sh->u_full[q]);
                }
                __syncwarp();
            }
            if (sh->abort_flag) {  // copies in flight land before the shared memory goes away
                for (uint32_t x = b > b_beg + KT_BLOCKS ? b - KT_BLOCKS : b_beg; x < b; x++) {
                    const uint32_t q = (x - b_0) % KT_BLOCKS, before = (x - b_0) / KT_BLOCKS - (b_0 + q < b_beg ? 1 : 0);
                    kt_wait(&sh->u_full[q], before & 1, sh, a.status, false);
                }
            }
        } else if (warp < 18) {
            // ---------------- instructions ----------------
            constexpr uint32_t idesc_qk = (1u << 4) | ((KT_TILE / 2 >> 3) << 17) | ((KT_TILE >> 4) << 24);
            constexpr uint32_t idesc_pv = (1u << 4) | ((HD >> 3) << 17) | ((KT_TILE >> 4) << 24);
            const int w = warp - 16;
            const uint64_t qd = smem_desc_sw128(smem_u32(smem + L::Q) + w * L::TILE), kd = smem_desc_sw128(smem_u32(smem + L::K)), vd = smem_desc_sw128(smem_u32(smem + L::V));
            const uint32_t s_at = tmem + w * KT_TILE, o_at = tmem + 2 * KT_TILE + w * HD;
            auto scores = [&](int slot, int h) {  // of a half of a tile's keys
                if (elect_one()) {
                    const uint64_t k = kd + ((slot * L::TILE + h * (HALF / 2)) >> 4);
#pragma unroll
                    for (int kk = 0; kk < HD / 16; kk++) {
                        const uint32_t at = (uint32_t)(kk >> 2) * (HALF >> 4) + 2 * (kk & 3);
                        mma_f16(s_at + 64 * h, qd + at, k + at, idesc_qk, kk > 0);
                    }
                    mma_commit(&sh->s_full[w][h]);
                    if (!h) mma_commit(&sh->k_empty[slot]);
                }
                __syncwarp();
            };
            bool ok = n > 0 && w < tiles;
            auto wait = [&](uint64_t* bar, uint32_t phase) {
                ok = ok && __all_sync(0xffffffffu, kt_wait(bar, phase, sh, a.status));
                tc_fence_after();
                return ok;
            };
            if (ok && wait(&sh->q_full, 0) && wait(&sh->k_full[0], 0)) {
                scores(0, 1);
                scores(0, 0);
            }
            for (int i = 0; i < n && ok; i++) {
                const int slot = i & 1, next = slot ^ 1;
                // The next tile's second half of the keys while this one's exponentials are made: probabilities take the first half's place.
                if (i + 1 < n) {
                    if (!wait(&sh->s_free[w], (uint32_t)(i & 1)) || !wait(&sh->k_full[next], (uint32_t)(((i + 1) >> 1) & 1))) break;
                    scores(next, 1);
                }
                if (!wait(&sh->v_full[slot], (uint32_t)((i >> 1) & 1))) break;
#pragma unroll
                for (int h = 0; h < 2; h++) {  // (the first half's products run under the second half's exponentials)
                    if (!wait(&sh->p_full[w][h], (uint32_t)(i & 1))) break;
                    if (elect_one()) {
                        const uint64_t v = vd + ((slot * L::TILE + h * VHALF) >> 4);
#pragma unroll
                        for (int kk = 0; kk < 4; kk++) kt_mma_ts(o_at, s_at + 32 * h + 8 * kk, v + 2 * kk, idesc_pv, (uint32_t)(i | h | kk));
                        if (h) mma_commit(&sh->v_empty[slot]);
                    }
                    __syncwarp();
                }
                if (ok && i + 1 < n) scores(next, 0);
            }
            // (a share without keys: its sums, zeros, take the queries' place, which other warps may still be writing)
            if (n == 0) kt_wait(&sh->q_full, 0, sh, a.status);
            if (elect_one()) mma_commit(&sh->o_full);
            __syncwarp();
            if (n > 0 && w < tiles && !ok) kt_wait(&sh->o_full, 0, sh, a.status, false);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 96;" ::: "memory");
        // ---------------- softmax ----------------
        // two warps a row: 0 .. 7 have the first and the third block of a tile's keys, 8 .. 15 the others
        const int w = (warp >> 2) & 1, hc = warp >> 3;
        const bool live = w < tiles;
        {  // the tile's queries as f16: sixteen rows a warp, a row's values over the lanes
            auto from = [&](uint32_t in_warp, uint32_t d) {
                const uint32_t r = min(r_block + w * KT_TILE + (warp & 3) * 32 + hc * 16 + in_warp, rows - 1), tok = kt_token(a, r);
                return (const T*)a.q + (size_t)(seq.r0 + tok) * a.q_stride + (size_t)(head * a.G + (r - tok * a.G)) * HD + d;
            };
            auto factor = [&](uint32_t row, uint32_t bits, bool first) {  // of a row whose largest magnitude has those bits (what is not finite is above all else)
                const int ex = min(max((int)(bits >> 23), 40), 254) - 127;
                if (first) sh->told[0][w * KT_TILE + row] = (bits >= 0x7f800000u ? NAN : pow2(ex)) * a.c2;
                return (ex == 127 ? 0x1p-127f : pow2(-ex)) * a.q_sign;  // (2^-127 has no exponent of its own: pow2 does not make it)
            };
            if (sizeof(T) == 2 && a.wide) {  // eight a lane: half the instructions of the form below
                constexpr int PER = HD / 8, ROWS = 32 / PER, FLIGHT = 16 / ROWS;
                const uint32_t d8 = (uint32_t)(lane % PER);
                uint8_t* const to = smem + L::Q + w * L::TILE + (d8 >> 3) * HALF;
#pragma unroll 1
                for (int i0 = 0; i0 < 16; i0 += FLIGHT * ROWS) {
                    uint4 eight[FLIGHT];
#pragma unroll
                    for (int i = 0; i < FLIGHT; i++) eight[i] = *(const uint4*)from((uint32_t)(i0 + i * ROWS + lane / PER), 8 * d8);
#pragma unroll
                    for (int i = 0; i < FLIGHT; i++) {
                        const uint32_t row = (uint32_t)((warp & 3) * 32 + hc * 16 + i0 + i * ROWS + lane / PER);
                        const T* const v = (const T*)&eight[i];
                        float x[8];
                        uint32_t bits = 0;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            x[e] = to_f32<T>(v[e]);
                            bits = max(bits, __float_as_uint(x[e]) & 0x7fffffffu);
                        }
#pragma unroll
                        for (int o = PER / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
                        const float f = factor(row, bits, d8 == 0);
                        *(uint4*)(to + row * 128 + (((d8 & 7) ^ (row & 7)) << 4)) =
                            make_uint4(kt_pack(x[0] * f, x[1] * f), kt_pack(x[2] * f, x[3] * f), kt_pack(x[4] * f, x[5] * f), kt_pack(x[6] * f, x[7] * f));
                    }
                }
            } else {
                constexpr int PER = HD / 4, ROWS = 32 / PER, FLIGHT = 8;
                const uint32_t d4 = (uint32_t)(lane % PER), half = d4 >> 4, chunk = (d4 & 15) >> 1, in = (d4 & 1) * 8;
#pragma unroll 1
                for (int i0 = 0; i0 < 16; i0 += FLIGHT * ROWS) {
                    float x[FLIGHT][4];
#pragma unroll
                    for (int i = 0; i < FLIGHT; i++) load4(x[i], from((uint32_t)(i0 + i * ROWS + lane / PER), 4 * d4), a.aligned);
#pragma unroll
                    for (int i = 0; i < FLIGHT; i++) {
                        const uint32_t row = (uint32_t)((warp & 3) * 32 + hc * 16 + i0 + i * ROWS + lane / PER);
                        uint32_t bits = 0;
#pragma unroll
                        for (int e = 0; e < 4; e++) bits = max(bits, __float_as_uint(x[i][e]) & 0x7fffffffu);
#pragma unroll
                        for (int o = PER / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
                        const float f = factor(row, bits, d4 == 0);
                        *(uint2*)(smem + L::Q + w * L::TILE + half * HALF + row * 128 + ((chunk ^ (row & 7)) << 4) + in) =
                            make_uint2(kt_pack(x[i][0] * f, x[i][1] * f), kt_pack(x[i][2] * f, x[i][3] * f));
                    }
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->q_full);
        }
        const uint32_t row = (uint32_t)((warp & 3) * 32 + lane), r = min(r_block + w * KT_TILE + row, rows - 1), tok = kt_token(a, r), qp = seq.start + tok;
        const uint32_t tile_qp = seq.start + kt_token(a, min(r_block + w * KT_TILE, rows - 1));                      // the tile's first position
        const uint32_t tile_end = seq.start + kt_token(a, min(r_block + w * KT_TILE + KT_TILE - 1, rows - 1));       // and its last
        const uint32_t see_to = max(qp + 1, prefix), my_lo = first_key(qp);                                           // keys my_lo .. see_to - 1
        const uint32_t all_to = max(tile_qp + 1, prefix), all_from = first_key(tile_end);
        bool ok = __all_sync(0xffffffffu, kt_wait(&sh->q_full, 0, sh, a.status));
        const float qf = sh->told[0][w * KT_TILE + row];
        // Both warps of a row: false when the CTA gives up. step: how often they have met.
        auto meet = [&](int step) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->pair[w][warp & 3]);
            return (bool)__all_sync(0xffffffffu, kt_wait(&sh->pair[w][warp & 3], (uint32_t)(step & 1), sh, a.status));
        };
        ok = ok && meet(0);
        const float slope = SPECIAL && a.slopes ? a.slopes[head * a.G + (r - tok * a.G)] * 1.44269504f : 0.0f;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16, s_at = tmem + lane_base + w * KT_TILE, o_at = tmem + lane_base + 2 * KT_TILE + w * HD;
        float m = -INFINITY, l = 0.0f;
        for (int i = 0; i < n && live && ok; i++) {
            uint32_t v[2][32];
            float f[2], mx[2];
            const uint32_t j0 = (b_0 + i * KT_BLOCKS + hc) * KV8_BLOCK;  // the warp's first key; its second block is 64 behind
            auto take = [&](const int h) {  // a block's scores, as far as they go without the row's largest
                ok = __all_sync(0xffffffffu, kt_wait(&sh->s_full[w][h], (uint32_t)(i & 1), sh, a.status));
                if (!ok) return;
                tc_fence_after();
                kt_ld32(s_at + 64 * h + 32 * hc, v[h]);
                const uint32_t bad = sh->bad[i & 3][2 * h + hc];
                // (not zero: a key that is not seen stays at -inf)
                f[h] = fmaxf(qf * sh->k_scale[i & 3][2 * h + hc], 1e-37f);
                if (qf != qf) f[h] = qf;
                kt_ld_wait();
                if (!h) {  // both are in registers
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh->s_free[w]);
                }
                if (SPECIAL) {
                    const float fh = f[h];
                    if (a.cap2 > 0.0f) {
                        // cap tanh(z), z = score / cap: by an odd polynomial fitted at Chebyshev nodes of z^2, off by 4.4e-7 up to |z| = 0.75, with the powers of what
                        // brings a score to z in its coefficients (below the smallest f32 they would add nothing: scores are below 2^15 here); beyond by exponentials
                        const float fz = fh * a.cap_z, fz2 = fz * fz;
                        float most = 0.0f;
#pragma unroll
                        for (int e = 0; e < 32; e += 2) most = max3(most, fabsf(__uint_as_float(v[h][e])), fabsf(__uint_as_float(v[h][e + 1])));
                        if (__any_sync(0xffffffffu, !(most * fz <= 0.75f) || fz > 1.0f)) {
#pragma unroll
                            for (int e = 0; e < 32; e++) {
                                const float z = __uint_as_float(v[h][e]) * fz, y = fabsf(z);
                                const float far = 1.0f - __fdividef(2.0f, 1.0f + kt_exp2(2.0f * 1.44269504f * y));
                                const float z2 = z * z;
                                const float near = y * fmaf(z2, fmaf(z2, fmaf(z2, fmaf(z2, K4, K3), K2), K1), K0);
                                v[h][e] = __float_as_uint(a.cap2 * copysignf(y > 0.75f ? far : near, z));
                            }
                        } else {
                            const float g0 = fz * a.cap2, g1 = g0 * fz2, g2 = g1 * fz2, g3 = g2 * fz2, g4 = g3 * fz2;
                            auto k = [](float x) { return make_float2(x, x); };
                            const float2 c0 = k(g0 * K0), c1 = k(g1 * K1), c2 = k(g2 * K2), c3 = k(g3 * K3), c4 = k(g4 * K4);
#pragma unroll
                            for (int e = 0; e < 32; e += 2) {
                                const float2 x = make_float2(__uint_as_float(v[h][e]), __uint_as_float(v[h][e + 1])), x2 = mul2(x, x);
                                const float2 y = mul2(x, fma2(x2, fma2(x2, fma2(x2, fma2(x2, c4, c3), c2), c1), c0));
                                v[h][e] = __float_as_uint(y.x);
                                v[h][e + 1] = __float_as_uint(y.y);
                            }
                        }
                        f[h] = 1.0f;
                    }
                    if (a.slopes) {
                        const float at = slope * (float)((int)(j0 + 64 * h) - (int)qp), g = f[h];
                        const float2 g2 = make_float2(g, g), s2 = make_float2(slope, slope), at2 = make_float2(at, at);
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const float2 bias = fma2(s2, make_float2((float)kt_tok(e), (float)kt_tok(e + 1)), at2);
                            const float2 y = fma2(make_float2(__uint_as_float(v[h][e]), __uint_as_float(v[h][e + 1])), g2, bias);
                            v[h][e] = __float_as_uint(y.x);
                            v[h][e + 1] = __float_as_uint(y.y);
                        }
                        f[h] = 1.0f;
                    }
                }
                if (bad) {
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        if (bad & (1u << kt_tok(e))) v[h][e] = 0x7fffffffu;
                }
                if (j0 + 64 * h + 32 > all_to || j0 + 64 * h < all_from) {  // some row does not see some key
                    auto below = [](uint32_t n, uint32_t from) { return n >= from + 32 ? 0xffffffffu : n <= from ? 0u : (1u << (n - from)) - 1; };  // a bit per key of the block below n
                    const uint32_t seen = below(see_to, j0 + 64 * h) & ~below(my_lo, j0 + 64 * h);
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        if (!(seen & (1u << kt_tok(e)))) v[h][e] = 0xff800000u;
                }
                mx[h] = fmaxf(__uint_as_float(v[h][0]), __uint_as_float(v[h][1]));
#pragma unroll
                for (int e = 2; e < 32; e += 2) mx[h] = max3(mx[h], __uint_as_float(v[h][e]), __uint_as_float(v[h][e + 1]));
                mx[h] *= f[h];
            };
            take(1);
            if (ok) take(0);
            if (!ok) break;
            // the row's other half (which has its scores, too, by then: probabilities take their place)
            sh->told[hc][w * KT_TILE + row] = fmaxf(mx[0], mx[1]);  // (the step ahead's has been read: its probabilities have been multiplied)
            tc_fence_before();
            ok = meet(i + 1);
            if (!ok) break;
            tc_fence_after();
            const float top = fmaxf(sh->told[0][w * KT_TILE + row], sh->told[1][w * KT_TILE + row]);
            if (i == 0) {
                m = top;
            } else if (__any_sync(0xffffffffu, top > m + LAZY_BITS)) {
                const float mn = fmaxf(m, top), g = m == -INFINITY ? 0.0f : kt_exp2(m - mn);
                m = mn;
                l *= g;
#pragma unroll 1
                for (int h = 0; h < HD / 16; h++) {  // (the warp's half of the dimensions, eight at a time: its scores are in registers)
                    uint32_t o[8];
                    const uint32_t at = o_at + hc * (HD / 2) + 8 * h;
                    kt_ld8(at, o);
                    kt_ld_wait();
#pragma unroll
                    for (int e = 0; e < 8; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * g);
                    kt_st8(at, o);
                }
            }
            const float base = m == -INFINITY ? 0.0f : KT_P_BITS - m;
            float2 part[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
            if (tiles == 2 && (w == 1 || i > 0)) {
                ok = __all_sync(0xffffffffu, kt_wait(&sh->turn[w], (uint32_t)((w == 1 ? i : i - 1) & 1), sh, a.status));
                if (!ok) break;
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t pk[16];
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const float g = f[h];
                    float2 x = fma2(make_float2(__uint_as_float(v[h][2 * e]), __uint_as_float(v[h][2 * e + 1])), make_float2(g, g), make_float2(base, base));
                    x = make_float2(kt_exp2(x.x), kt_exp2(x.y));
                    part[e & 1] = add2(part[e & 1], x);
                    pk[e] = kt_pack(x.x, x.y);
                }
                kt_st16(s_at + 32 * h + 16 * hc, pk);
                if (h && tiles == 2 && lane == 0) mbar_arrive(&sh->turn[w ^ 1]);
                kt_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh->p_full[w][h]);
            }
            l += (part[0].x + part[0].y) + (part[1].x + part[1].y);
        }
        // ---------------- the sums, into shared memory over queries and keys, their largest scores and denominators over the values ----------------
        float2* const ml = (float2*)(smem + L::V);
        ok = __all_sync(0xffffffffu, kt_wait(&sh->o_full, 0, sh, a.status) && !sh->abort_flag);
        if (ok && live) {
            tc_fence_after();
            if (sh->far) {
                far_sums<HD, SPECIAL, T>(a, sh, w * KT_TILE + (warp & 3) * 32 + hc * 16, __shfl_sync(0xffffffffu, m, (lane & 15) + hc * 16), (float*)(smem + L::RING) + warp * HD, smem, ml);
            } else {
                float4* const dst = (float4*)(smem + (size_t)(w * KT_TILE + row) * HD * 4);
                const float one = __uint_as_float(*(volatile uint32_t*)&sh->v_top) * (KT_SUM_DOWN / V_ONE);
#pragma unroll
                for (int h = hc * (HD / 64); h < (hc + 1) * (HD / 64); h++) {
                    uint32_t o[32];
                    kt_ld32(o_at + 32 * h, o);
                    kt_ld_wait();
                    auto f = [&](int e) { return n > 0 ? __uint_as_float(o[e]) * one : 0.0f; };
#pragma unroll
                    for (int e = 0; e < 8; e++) dst[(8 * h + e) ^ (row & 7)] = make_float4(f(4 * e), f(4 * e + 1), f(4 * e + 2), f(4 * e + 3));
                }
                sh->told[hc][w * KT_TILE + row] = l;
                if (meet(n + 1) && hc == 0) {
                    l += sh->told[1][w * KT_TILE + row];
                    ml[w * KT_TILE + row] = make_float2(m, a.Z > 1 ? l : l > 0.0f || l != l ? KT_SUM_UP / l : 0.0f);
                }
            }
        }
        __syncwarp();
        if (a.Z > 1) cluster_sync_all();
        else asm volatile("bar.sync 1, 512;" ::: "memory");
        // ---------------- the rows out: CTA z every Z-th run of them ----------------
        if (!sh->abort_flag) {
            constexpr int PER = HD / 4, ROWS = 32 / PER;
            const uint32_t f4 = (uint32_t)(lane % PER), count = r_end - r_block;
            auto put = [&](uint32_t at, float4 o, float inv) {
                const uint32_t rr = r_block + at, tk = kt_token(a, rr);
                kt_store4<T>((T*)a.out + (size_t)(seq.r0 + tk) * a.out_stride + (size_t)(head * a.G + (rr - tk * a.G)) * HD + 4 * f4,
                             make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv), a.aligned);
            };
            auto from_of = [&](uint32_t at) { return (const float4*)(smem + (size_t)at * HD * 4) + (f4 ^ (at & 7)); };
            if (sizeof(T) == 2 && a.Z == 1 && a.wide) {
                constexpr uint32_t PER8 = HD / 8, ROWS8 = 32 / PER8;
                const uint32_t d8 = (uint32_t)lane % PER8;
#pragma unroll 4
                for (uint32_t at = warp * ROWS8 + lane / PER8; at < count; at += 16 * ROWS8) {
                    const float4* const row = (const float4*)(smem + (size_t)at * HD * 4);
                    const float4 x = row[(2 * d8) ^ (at & 7)], y = row[(2 * d8 + 1) ^ (at & 7)];
                    const float inv = ml[at].y, v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
                    const uint32_t rr = r_block + at, tk = kt_token(a, rr);
                    alignas(16) T o[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        if constexpr (std::is_same<T, __half>::value) o[e] = __float2half_rn(v[e] * inv);
                        else o[e] = (T)(v[e] * inv);  // (to nearest even)
                    }
                    *(uint4*)((T*)a.out + (size_t)(seq.r0 + tk) * a.out_stride + (size_t)(head * a.G + (rr - tk * a.G)) * HD + 8 * d8) = *(const uint4*)o;
                }
            } else if (a.Z == 1) {
#pragma unroll 4
                for (uint32_t at = warp * ROWS + lane / PER; at < count; at += 16 * ROWS) put(at, *from_of(at), ml[at].y);
            } else {
                for (uint32_t at = (z * 16 + warp) * ROWS + lane / PER; at < count; at += a.Z * 16 * ROWS) {
                    const float4* const from = from_of(at);
                    float4 o;
                    float den;
                    float2 p[8];
                    float4 b[8];
                    float M = -INFINITY;
#pragma unroll
                    for (uint32_t k = 0; k < 8; k++) {  // (Z is 2, 4 or 8)
                        if (k >= a.Z) break;
                        p[k] = kt_peer_f2(ml + at, k);
                        b[k] = kt_peer_f4(from, k);
                        M = fmaxf(M, p[k].x);
                    }
                    o = make_float4(0.f, 0.f, 0.f, 0.f);
                    den = 0.0f;
#pragma unroll
                    for (uint32_t k = 0; k < 8; k++) {
                        if (k >= a.Z) break;
                        const float g = p[k].x == -INFINITY ? p[k].y : kt_exp2(p[k].x - M);  // (a share that sees nothing: zero, or NaN where its keys are)
                        o = make_float4(fmaf(g, b[k].x, o.x), fmaf(g, b[k].y, o.y), fmaf(g, b[k].z, o.z), fmaf(g, b[k].w, o.w));
                        den = fmaf(g, p[k].y, den);
                    }
                    put(at, o, den > 0.0f || den != den ? KT_SUM_UP / den : 0.0f);
                }
            }
        }
    }
    if (a.Z > 1) {  // no CTA leaves while another reads its sums
        if (warp >= 16) cluster_sync_all();
        cluster_sync_all();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(KT_TMEM_COLS) : "memory");
    }
}

template <int HD, bool SPECIAL, typename T>
cudaError_t rows_t(KtArgs& a, cudaStream_t st, bool pdl) {
    constexpr size_t smem = KtSizes<HD>::BYTES;
    auto kern = attend_kv8_rows_kernel<HD, SPECIAL, T>;
    if (cudaError_t e = ensure_dynamic_smem((const void*)kern, smem, 0); e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.blocks * a.c.nkv * a.Z);
    cfg.blockDim = dim3(KT_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.Z;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}
template <int HD, typename T>
cudaError_t rows_s(KtArgs& a, cudaStream_t st, bool pdl) {
    return a.cap2 > 0.0f || a.slopes ? rows_t<HD, true, T>(a, st, pdl) : rows_t<HD, false, T>(a, st, pdl);
}
template <int HD>
cudaError_t rows_hd(KtArgs& a, int dtype, cudaStream_t st, bool pdl) {
    switch (dtype) {
        case B2_F32: return rows_s<HD, float>(a, st, pdl);
        case B2_F16: return rows_s<HD, __half>(a, st, pdl);
        case B2_BF16: return rows_s<HD, __nv_bfloat16>(a, st, pdl);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

// Blocks of 256 rows: those of all sequences together are at most one a sequence more than of as many rows in a row.
static size_t kv8_row_blocks(const Kv8Seqs& s, uint32_t G) {
    const size_t rows = (size_t)s.n_rows * G;
    return s.n_seqs == 1 ? (rows + 2 * KT_TILE - 1) / (2 * KT_TILE) : rows / (2 * KT_TILE) + s.n_seqs;
}
// A grid of at most 2^31 CTAs, shares of the keys included; rows times heads a KV head stay exact through g_inv.
bool attend_kv8_rows_supports(const Kv8Cache& c, const Kv8Seqs& s, uint32_t nh) {
    const size_t G = nh / c.nkv;
    return kv8_row_blocks(s, (uint32_t)G) * c.nkv <= 0x7fffffffu / 8 && s.n_rows * G <= 0x7fffffffu / G;
}

cudaError_t launch_attend_kv8_rows(const Kv8Cache& c, const Kv8Seqs& s, const Kv8Attn& p, const void* q, size_t q_stride, void* out, size_t out_stride, int dtype,
                                   uint32_t* status, cudaStream_t st, bool pdl) {
    if (!kv8_supports(c.nkv, c.hd) || p.nh == 0 || p.nh % c.nkv) return cudaErrorInvalidValue;
    if (s.n_seqs == 0 || s.n_rows == 0 || s.max_rows == 0) return cudaSuccess;
    KtArgs a{};
    a.c = c;
    a.sq = s;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.G = p.nh / c.nkv;
    a.g_inv = a.G == 1 ? 0u : (uint32_t)(((1ull << 32) + a.G - 1) / a.G);
    if (!attend_kv8_rows_supports(c, s, p.nh)) return cudaErrorInvalidValue;
    const size_t blocks = kv8_row_blocks(s, a.G);
    a.blocks = (uint32_t)blocks;
    a.Z = 1;
    // Shares of the keys while two fit the chip beside each other (of clusters of eight no more than fourteen do) and have two tiles each. 32 heads of 8 KV heads of 128
    // behind 4096 keys, us without and with: 64 tokens 110 / 24, 512 tokens (64 CTAs) 81 / 49.
    while (a.Z < 8 && 2 * a.Z * blocks * c.nkv <= (a.Z == 4 ? 112 : 148) && 4 * a.Z * KT_BLOCKS <= s.max_blocks) a.Z *= 2;
    a.window = p.window <= 0x7fffffffu ? p.window : 0;
    a.q_sign = p.scale < 0.0f ? -1.0f : 1.0f;
    a.c2 = p.scale * a.q_sign * 1.44269504f;
    a.cap2 = p.cap * 1.44269504f;
    a.cap_z = p.cap > 0.0f ? 0.69314718f / p.cap : 0.0f;
    a.slopes = p.slopes;
    a.prefix = p.prefix;
    a.status = status;
    const size_t esz = dtype == B2_F32 ? 4 : 2, unit = 4 * esz;
    a.aligned = (((uintptr_t)q | (uintptr_t)out | q_stride * esz | out_stride * esz) & (unit - 1)) == 0;
    a.wide = (((uintptr_t)q | (uintptr_t)out | q_stride * esz | out_stride * esz) & 15) == 0;
    return c.hd == 64 ? rows_hd<64>(a, dtype, st, pdl) : rows_hd<128>(a, dtype, st, pdl);
}

}  // namespace b2
