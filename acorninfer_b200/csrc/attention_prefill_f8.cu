// Prefill attention over the pages of the 8-bit cache (f8_cache.cuh) on the 5th-generation tensor cores, head sizes 64 and 128:
// causal attention of a tile of 128 consecutive queries of one request, S = Q K^T and O += P V by tcgen05.mma with the
// accumulators in tensor memory.
//
// One CTA per (tile of 128 queries, pair of query heads that share a key/value head), one CTA to an SM, as in
// attention_prefill_tc.cu: the two heads ("units") read the same tiles and take turns on the tensor cores.  What is new is that K
// and V arrive as codes and are turned into bfloat16 on the way, which is exact (code * 2^e is a bfloat16 number), so that the
// products are those of a bfloat16 cache of the same numbers.  Why not 8-bit matrix instructions: the queries and the weights
// would have to be cut into e4m3 parts, two at least, and a product would take as long as one in bfloat16.
//   warps 0-3  softmax of unit 0, warps 4-7 of unit 1: thread r owns query row r (= TMEM lane r): masks, exponentiates
//              in float32 base 2 against a reference maximum that moves when a row outgrew it by 2^8, writes P (bfloat16) over S.
//   warps 8-11 turn a block's codes into the operand tiles, 32 keys a warp: 16 codes a lane (16 bytes in, 32 out, swizzled as the
//              matrix instruction wants them).  s eeee mmm shifted into a bfloat16 number's places reads 2^-120 times its value,
//              subnormal codes included; one multiplication by 2^(120 + e) makes it the entry (a second one where e > 7).
//              Keys that no query of the tile reads get zero values (a slot that was never written may hold anything);
//              a row that is no number gets a NaN key, which spoils the queries that read it, and zero values.
//   warp 12    producer: TMA loads of Q (once) and of the codes of each block of 128 keys (a box is the keys and the values of one
//              page and head), asynchronous copies of their exponents, into two stages of 32 KB.
//   warp 13    MMA issuer (converged; one elected lane issues): per block j and unit u, O_u += P_u[j] V_j with P from
//              tensor memory, then S_u = Q_u K_{j+1}^T into the columns P_u[j] was read from.
// The softmax warps need 184 registers a thread, sixteen warps get 128 each: the warpgroups share 4 x 128 out as 184, 184,
// 80 (codes) and 64 (the rest).  Operand tiles K_0 V_0 K_1 V_1 ... go through a ring of three.  Tensor memory (512 columns): S / P of unit u at columns 128 u,
// O of unit u at 256 + 128 u.
//
// Every mbarrier wait is bounded; a wait that gives up records g_attn_pre_f8_error and the CTA drains.
#include "f8_tma.cuh"

#define PF8_BM 128
#define PF8_BN 128
#define PF8_SLOTS 3
#define PF8_STAGES 2
#define PF8_THREADS 512               // two of the 16 warps are there for the register split, which goes by warpgroups
#define PF8_RESCALE_LOG2 8.0f
#define PF8_TMEM_COLS 512

__device__ int g_attn_pre_f8_error = 0;

struct PrefillF8Params {
    F8AttnParams a;
    int pairs, joint, v_first;       // pairs = ceil((nq / nkv) / 2): CTAs per (tile, kv head)
};

template <int D> struct PrefillF8 {
    static constexpr int HALVES = D / 64;
    static constexpr int HALF_BYTES = PF8_BN * 128;                  // [128 rows x 64 entries] bf16
    static constexpr int Q_BYTES = HALVES * PF8_BM * 128;            // one unit
    static constexpr int TILE_BYTES = HALVES * HALF_BYTES;           // a K or V operand tile
    static constexpr int RAW_BYTES = 2 * PF8_BN * D;                 // the codes of a block's keys and values
    static constexpr int SCALE_BYTES = 2 * PF8_BN;
    static constexpr int TILES = 2 * Q_BYTES;                        // offsets in shared memory
    static constexpr int RAW = TILES + PF8_SLOTS * TILE_BYTES;
    static constexpr int SCALES = RAW + PF8_STAGES * RAW_BYTES;
    static constexpr int BARS = SCALES + PF8_STAGES * SCALE_BYTES;
    // q_full, raw_full, raw_empty [STAGES], full, empty [SLOTS], s_full, p_full, o_done [unit]
    static constexpr int NUM_BARS = 1 + 2 * PF8_STAGES + 2 * PF8_SLOTS + 6;
    static constexpr int SMEM = BARS + NUM_BARS * 8 + 16;
};

__device__ __forceinline__ void pf8_mask(float (&s)[64], int key0, int qpos, bool row_ok, int first_seen, int keep) {
#pragma unroll
    for (int c = 0; c < 64; ++c) {
        const int key = key0 + c;
        const bool seen = key <= qpos && row_ok && (key >= first_seen || key < keep);
        s[c] = seen ? s[c] : -INFINITY;
    }
}

__device__ __forceinline__ float pf8_max(const float (&s)[64]) {
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < 64; c += 4) {
        m[0] = fmaxf(m[0], s[c]); m[1] = fmaxf(m[1], s[c + 1]);
        m[2] = fmaxf(m[2], s[c + 2]); m[3] = fmaxf(m[3], s[c + 3]);
    }
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// w[i] = bf16x2(2^((s[2i] - ref) * scale), 2^((s[2i+1] - ref) * scale)); returns the sum of the 64 values.  The rounding of
// ref * scale is a factor that all weights of a row share; where it could be a large one (scores beyond 2^20), the
// difference is taken first.
__device__ __forceinline__ float pf8_exp_pack(float (&s)[64], float scale_log2, float ref, uint32_t (&w)[32]) {
    float ps[4] = {0.f, 0.f, 0.f, 0.f};
    float neg_ref = -(ref * scale_log2);
    if (__any_sync(0xffffffffu, fabsf(neg_ref) > 1048576.f)) {
#pragma unroll
        for (int c = 0; c < 64; ++c) s[c] -= ref;
        neg_ref = 0.f;
    }
#pragma unroll
    for (int c = 0; c < 64; c += 2) {
        const float a = fast_exp2(fmaf(s[c], scale_log2, neg_ref));
        const float b = fast_exp2(fmaf(s[c + 1], scale_log2, neg_ref));
        ps[(c >> 1) & 3] += a + b;
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        w[c >> 1] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return (ps[0] + ps[1]) + (ps[2] + ps[3]);
}

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Two neighbouring codes (bytes `sel` and `sel` + 1 of w) as bfloat16 numbers times 2^-120.
template <int SEL> __device__ __forceinline__ uint32_t codes_to_bf16x2(uint32_t w) {
    const uint32_t x = __byte_perm(w, 0u, SEL == 0 ? 0x1404 : 0x3424);       // each code in the high byte of its half
    return ((x >> 4) & 0x07f007f0u) | (x & 0x80008000u);
}

template <int D>
__global__ void __launch_bounds__(PF8_THREADS, 1) attention_prefill_f8_kernel(const __grid_constant__ CUtensorMap map_q,
                                                                              const __grid_constant__ CUtensorMap map_k,
                                                                              const __grid_constant__ CUtensorMap map_v,
                                                                              const PrefillF8Params pp) {
    using L = PrefillF8<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const F8AttnParams& p = pp.a;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
    const uint32_t q_full = tc_smem(bars);
    const uint32_t raw_full0 = q_full + 8, raw_empty0 = raw_full0 + 8 * PF8_STAGES;
    const uint32_t full0 = raw_empty0 + 8 * PF8_STAGES, empty0 = full0 + 8 * PF8_SLOTS;
    const uint32_t s_full0 = empty0 + 8 * PF8_SLOTS, p_full0 = s_full0 + 16, o_done0 = p_full0 + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::NUM_BARS);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // CTAs are started in the order of the tile list; CTAs next to one another share a tile and mostly a key/value head.
    const int per_tile = p.nkv * pp.pairs;
    const int tile = (int)(blockIdx.x / per_tile);
    const int kvh = (int)(blockIdx.x % per_tile) / pp.pairs, pair = (int)(blockIdx.x % per_tile) % pp.pairs;
    const int rep = p.nq / p.nkv;
    const int head0 = kvh * rep + 2 * pair;
    const int units = (2 * pair + 1 < rep) ? 2 : 1;
    if (tc_smem(smem) & 1023u) {            // the swizzled tiles need a 1024-byte aligned base
        if (threadIdx.x == 0) tc_fail(&g_attn_pre_f8_error, 9, ACORN_KERNEL_ATTN_PREFILL_F8);
        return;
    }
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int s = 0; s < PF8_STAGES; ++s) { mbar_init(raw_full0 + 8 * s, 33); mbar_init(raw_empty0 + 8 * s, 4); }
        for (int s = 0; s < PF8_SLOTS; ++s) { mbar_init(full0 + 8 * s, 4); mbar_init(empty0 + 8 * s, 1); }
        for (int u = 0; u < 2; ++u) { mbar_init(s_full0 + 8 * u, 1); mbar_init(p_full0 + 8 * u, 4); mbar_init(o_done0 + 8 * u, 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 13) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(tc_smem(tmem_slot)), "r"((uint32_t)PF8_TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t tmem_s = tmem_base, tmem_o = tmem_base + 256;

    pdl_wait();
    pdl_trigger();
    const int r = p.tiles[2 * tile], q0 = p.tiles[2 * tile + 1];
    const int tok0 = p.row_start[r] + q0;
    const int n_q = min(PF8_BM, p.row_start[r + 1] - tok0);
    const int pos0 = p.row_pos[r] + q0;
    const int hi = pos0 + n_q;                                           // keys < hi are read by the tile
    const int lo_seen = mask_lo(p.mask, pos0);                           // the first query's rule starts first
    const int lo = lo_seen & ~(PF8_BN - 1);                              // blocks start at multiples of 128 keys
    // the kept first keys, where the rule's range starts beyond them, are nkb blocks of their own in front
    const int nkb = (p.mask.keep > 0 && lo > 0) ? min((p.mask.keep + PF8_BN - 1) / PF8_BN, lo / PF8_BN) : 0;
    const int nb = n_q > 0 ? nkb + (hi - lo + PF8_BN - 1) / PF8_BN : 0;
    auto key0_of = [&](int j) { return j < nkb ? j * PF8_BN : lo + (j - nkb) * PF8_BN; };
    const int log_box = min(p.logP, 7), box = 1 << log_box;

    if (warp >= 12) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
      if (warp == 12) {
        // ---------------------------------------------------------------- producer
        // The whole warp: lane l looks up the cache row of keys 4 l .. 4 l + 3 of a block, a block ahead of the loads, and copies
        // their exponents; an elected lane issues the boxes (one page, or 128 keys of a larger one).
        if (nb > 0 && elect_one()) {
            mbar_expect_tx(q_full, units * L::Q_BYTES);
            for (int u = 0; u < units; ++u)
                for (int h = 0; h < L::HALVES; ++h)
                    tma_load_2d(tc_smem(smem) + u * L::Q_BYTES + h * PF8_BM * 128, &map_q, q_full, (head0 + u) * D + 64 * h, tok0);
        }
        const int* table = p.block_table + (int64_t)r * p.table_stride - p.page_base[r];
        const int first_key = p.page_base[r] << p.logP;
        auto row_at = [&](int j) -> int {
            const int key = key0_of(j) + 4 * lane;
            int b = key & ~(box - 1);
            if (b >= hi) b = (hi - 1) & ~(box - 1);                      // masked later: any box that exists
            if (b < first_key) b = first_key;
            const int page = table[b >> p.logP];
            return ((page * p.nkv + kvh) << p.logP) + (b & ((1 << p.logP) - 1)) + (key & (box - 1));
        };
        int row_next = nb > 0 ? row_at(0) : 0;
        for (int j = 0; j < nb; ++j) {
            const int row = row_next, s = j % PF8_STAGES;
            if (j + 1 < nb) row_next = row_at(j + 1);
            const bool got = mbar_wait(raw_empty0 + 8 * s, ((j / PF8_STAGES) & 1) ^ 1);
            if (!got && lane == 0) tc_fail(&g_attn_pre_f8_error, 1, ACORN_KERNEL_ATTN_PREFILL_F8);
            if (!__all_sync(0xffffffffu, got)) break;
            if (elect_one()) mbar_expect_tx(raw_full0 + 8 * s, L::RAW_BYTES);
            cp_async_bytes<8>(tc_smem(smem + L::SCALES + s * L::SCALE_BYTES) + 8 * lane, p.scales + 2 * (int64_t)row);
            cp_async_arrive(raw_full0 + 8 * s);
            for (int k = 0; k < PF8_BN; k += box) {
                const int y = __shfl_sync(0xffffffffu, row, k >> 2);
                if (elect_one()) {
                    const uint32_t dst = tc_smem(smem + L::RAW + s * L::RAW_BYTES) + (uint32_t)(2 * k * D);
                    tma_load_3d(dst, &map_k, raw_full0 + 8 * s, 0, y, 0);
                    if (!pp.joint) tma_load_3d(dst + box * D, &map_v, raw_full0 + 8 * s, 0, y, 0);
                }
            }
        }
      } else if (warp == 13) {
        // ---------------------------------------------------------------- MMA issuer
        constexpr uint32_t IDESC_QK = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(PF8_BN >> 3) << 17) |
                                      ((uint32_t)(PF8_BM >> 4) << 24);
        constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) |
                                      ((uint32_t)(D >> 3) << 17) | ((uint32_t)(PF8_BM >> 4) << 24);
        auto wait_all = [&](uint32_t bar, uint32_t parity, int code) -> bool {
            const bool ok = mbar_wait(bar, parity);
            if (!ok && lane == 0) tc_fail(&g_attn_pre_f8_error, code, ACORN_KERNEL_ATTN_PREFILL_F8);
            return __all_sync(0xffffffffu, ok);
        };
        const uint32_t qlo = umma_lo(tc_smem(smem)), klo0 = umma_lo(tc_smem(smem + L::TILES));
        const uint32_t vlo0 = umma_lo_mn(tc_smem(smem + L::TILES), L::HALF_BYTES);
        auto issue_qk = [&](int u, int slot) {                          // S_u = Q_u K^T, K in `slot`
            const uint32_t klo = klo0 + slot * (L::TILE_BYTES >> 4);
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
                umma_bf16_elect(tmem_s + u * 128, qlo + ((u * L::Q_BYTES + (k >> 2) * PF8_BM * 128) >> 4) + 2 * (k & 3),
                                klo + (((k >> 2) * L::HALF_BYTES) >> 4) + 2 * (k & 3), IDESC_QK, k > 0 ? 1u : 0u);
            umma_commit_elect(s_full0 + 8 * u);
        };
        bool good = nb > 0 && wait_all(q_full, 0, 2);
        int slot = 0, phase = 0;                                         // the next tile of the ring
        if (good) {
            good = wait_all(full0, 0, 3);
            tc_fence_after();
            if (good) {
                for (int u = 0; u < units; ++u) issue_qk(u, 0);
                umma_commit_elect(empty0);
                slot = 1;
            }
        }
        for (int j = 0; j < nb && good; ++j) {
            const int sv = slot, pv = phase;                             // V_j
            if (++slot == PF8_SLOTS) { slot = 0; phase ^= 1; }
            const int sk = slot, pk = phase;                             // K_{j+1}
            const bool has_next = j + 1 < nb;
            if (has_next) { if (++slot == PF8_SLOTS) { slot = 0; phase ^= 1; } }
            good = wait_all(full0 + 8 * sv, pv, 3);
            if (!good) break;
            const uint32_t vlo = vlo0 + sv * (L::TILE_BYTES >> 4);
            for (int u = 0; u < units && good; ++u) {
                good = wait_all(p_full0 + 8 * u, j & 1, 4);
                if (!good) break;
                tc_fence_after();
                // 16 keys a step: P advances 8 columns, V 16 rows of 128 bytes
#pragma unroll
                for (int k = 0; k < PF8_BN / 16; ++k)
                    umma_bf16_ts_elect(tmem_o + u * 128, tmem_s + u * 128 + 8 * k, vlo + ((k * 16 * 128) >> 4), IDESC_PV,
                                       k > 0 || j > 0 ? 1u : 0u);
                if (u == units - 1) umma_commit_elect(empty0 + 8 * sv);
                // the next scores go where P was: the pipe runs them after the product above
                if (has_next) {
                    if (u == 0) good = wait_all(full0 + 8 * sk, pk, 5);
                    if (good) issue_qk(u, sk);
                } else {
                    umma_commit_elect(o_done0 + 8 * u);
                }
            }
            if (good && has_next) umma_commit_elect(empty0 + 8 * sk);
        }
      }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        // ---------------------------------------------------------------- codes to operand tiles
        constexpr int PIECES = D / 16, KEYS = 32 / PIECES;               // 16-byte pieces of a row; keys the warp takes at a time
        const int w0 = (warp - 8) * 32;
        const int piece = lane % PIECES, sub = lane / PIECES;
        const int chunk0 = (2 * piece) & 7;                              // the first of the piece's two 16-byte chunks in its half
        const int half_off = (piece >> 2) * L::HALF_BYTES;
        // (lanes of the second half write their second chunk first: the two halves' chunks then lie in different banks)
        const int swap = D == 128 ? piece >> 2 : 0;
        int slot = 0, phase = 0;
        for (int j = 0; j < nb; ++j) {
            const int s = j % PF8_STAGES;
            bool got = mbar_wait(raw_full0 + 8 * s, (j / PF8_STAGES) & 1);
            if (!got) tc_fail(&g_attn_pre_f8_error, 11, ACORN_KERNEL_ATTN_PREFILL_F8);
            if (!__all_sync(0xffffffffu, got)) break;
            const uint32_t bytes = *reinterpret_cast<const uint16_t*>(smem + L::SCALES + s * L::SCALE_BYTES + 2 * (w0 + lane));
            const int kbyte = bytes & 255u, vbyte = bytes >> 8, key = key0_of(j) + w0 + lane;
            const bool read = key < hi && (key >= lo_seen || key < p.mask.keep);
            bool fine = true;
            for (int kv = 0; kv < 2; ++kv) {
                // this lane's key: 2^(120 + e) = 2^(byte - 7), as two factors where that is beyond bfloat16
                const int byte = kv ? vbyte : kbyte;
                const bool none = kbyte == F8_NAN_BYTE || vbyte == F8_NAN_BYTE;
                const bool large = byte > 134;
                uint32_t f1 = (uint32_t)(large ? 127 + 120 : byte + 120) << 7, f2 = large ? (uint32_t)byte << 7 : 0x3f80u;
                if (none) { f1 = kv ? 0u : 0x7fc0u; f2 = 0x3f80u; }
                if (kv && !read) { f1 = 0u; f2 = 0x3f80u; }
                const bool any_large = __any_sync(0xffffffffu, f2 != 0x3f80u);
                const uint32_t both = f1 | f2 << 16;
                got = mbar_wait(empty0 + 8 * slot, phase ^ 1);
                if (!got) tc_fail(&g_attn_pre_f8_error, 12, ACORN_KERNEL_ATTN_PREFILL_F8);
                fine = __all_sync(0xffffffffu, got);
                if (!fine) break;
                const uint8_t* raw = smem + L::RAW + s * L::RAW_BYTES;
                uint8_t* tile_at = smem + L::TILES + slot * L::TILE_BYTES + half_off;
                const int skip = (kv ^ pp.v_first) << log_box;           // the values' rows follow the keys', or the other way round
#pragma unroll 4
                for (int it = 0; it < 32 / KEYS; ++it) {
                    const int k = it * KEYS + sub;
                    const uint4 c = *reinterpret_cast<const uint4*>(raw + (f8_stage_row(w0 + k, log_box) + skip) * D + 16 * piece);
                    const uint32_t f = __shfl_sync(0xffffffffu, both, k);
                    const uint32_t fa = __byte_perm(f, 0u, 0x1010), fb = __byte_perm(f, 0u, 0x3232);
                    const uint32_t cw[4] = {c.x, c.y, c.z, c.w};
                    uint32_t v[8];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        v[2 * q] = mul_bf16x2(codes_to_bf16x2<0>(cw[q]), fa);
                        v[2 * q + 1] = mul_bf16x2(codes_to_bf16x2<2>(cw[q]), fa);
                    }
                    if (any_large) {
#pragma unroll
                        for (int q = 0; q < 8; ++q) v[q] = mul_bf16x2(v[q], fb);
                    }
                    const int row = w0 + k;
                    uint8_t* at = tile_at + row * 128;
                    const uint4 lo4 = make_uint4(v[0], v[1], v[2], v[3]), hi4 = make_uint4(v[4], v[5], v[6], v[7]);
                    *reinterpret_cast<uint4*>(at + (((chunk0 + swap) ^ (row & 7)) << 4)) = swap ? hi4 : lo4;
                    *reinterpret_cast<uint4*>(at + (((chunk0 + 1 - swap) ^ (row & 7)) << 4)) = swap ? lo4 : hi4;
                }
                fence_proxy_async();                                     // the matrix instructions read what was written here
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(full0 + 8 * slot);
                    if (kv) mbar_arrive(raw_empty0 + 8 * s);
                }
                if (++slot == PF8_SLOTS) { slot = 0; phase ^= 1; }
            }
            if (!fine) break;
        }
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
      if (warp < 4 * units) {
        // ---------------------------------------------------------------- softmax and output
        const int u = warp >> 2;
        const int row = (warp & 3) * 32 + lane;                          // query row = TMEM lane
        const int head = head0 + u;
        const int qpos = pos0 + row;
        const int first_seen = mask_lo(p.mask, qpos);
        const bool row_ok = row < n_q;
        const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t my_s = tmem_s + lane_addr + u * 128, my_o = tmem_o + lane_addr + u * 128;
        const uint32_t s_full = s_full0 + 8 * u, p_full = p_full0 + 8 * u, o_done = o_done0 + 8 * u;
        const int last_lo = n_q > 0 ? mask_lo(p.mask, hi - 1) : 0;       // the last query's rule starts last
        float m_ref = -INFINITY, ref = 0.f, l_run = 0.f;                 // the reference in units of log2, and of the scores
        bool good = nb > 0;
        for (int j = 0; j < nb; ++j) {
            // S of block j is complete; so is P V of block j-1, issued before it: O is stable
            if (!mbar_wait(s_full, j & 1)) { tc_fail(&g_attn_pre_f8_error, 6, ACORN_KERNEL_ATTN_PREFILL_F8); good = false; }
            good = __all_sync(0xffffffffu, good);
            if (!good) break;
            tc_fence_after();
            const int key0 = key0_of(j);
            // a block that every query of the tile sees whole needs no mask
            const bool masked = key0 + PF8_BN - 1 > pos0 || key0 < last_lo || n_q < PF8_BM;
            // One pass in the common case: exponentiate against the reference maximum the row already has while the block's own
            // maximum is taken; only a row whose maximum outgrew the reference by more than 2^8 (always so in its first
            // block) moves the reference, and then the warp reads the block again.
            float s[64];
            uint32_t w_lo[32], w_hi[32];
            tmem_ld64(my_s, s);
            if (masked) pf8_mask(s, key0, qpos, row_ok, first_seen, p.mask.keep);
            float mx = pf8_max(s);
            float psum = pf8_exp_pack(s, p.scale_log2, ref, w_lo);
            tmem_ld64(my_s + 64, s);
            if (masked) pf8_mask(s, key0 + 64, qpos, row_ok, first_seen, p.mask.keep);
            const float top = fmaxf(mx, pf8_max(s));
            mx = top * p.scale_log2;                                     // the scale is positive
            float corr = 1.f;
            const bool grew = mx > m_ref + PF8_RESCALE_LOG2;
            if (__any_sync(0xffffffffu, grew)) {
                if (grew) {
                    corr = fast_exp2(m_ref - mx);                        // m_ref = -inf: 0
                    l_run *= corr;
                    m_ref = mx;
                    ref = top;
                }
                psum = pf8_exp_pack(s, p.scale_log2, ref, w_hi);
                tmem_ld64(my_s, s);
                if (masked) pf8_mask(s, key0, qpos, row_ok, first_seen, p.mask.keep);
                psum += pf8_exp_pack(s, p.scale_log2, ref, w_lo);
            } else {
                psum += pf8_exp_pack(s, p.scale_log2, ref, w_hi);
            }
            l_run += psum;
            if (j > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    float part[32];
                    tmem_ld32(my_o + c, part);
#pragma unroll
                    for (int i = 0; i < 32; ++i) part[i] *= corr;
                    tmem_st32(my_o + c, part);
                }
            }
            // P over the first 64 columns of S: column c holds keys 2c and 2c + 1
            tmem_st32_raw(my_s, w_lo);
            tmem_st32_raw(my_s + 32, w_hi);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full);
        }
        if (good) {
            if (!mbar_wait(o_done, 0)) { tc_fail(&g_attn_pre_f8_error, 8, ACORN_KERNEL_ATTN_PREFILL_F8); good = false; }
            good = __all_sync(0xffffffffu, good);
        }
        if (good) {
            tc_fence_after();
            // a sink is one more term of the denominator, against the same reference maximum as the keys' terms
            if (p.sink && row_ok) l_run += exp2f(p.sink[head] * 1.4426950408889634f - m_ref);
            const float inv = row_ok ? 1.f / l_run : 0.f;
            bf16* orow = p.out + ((int64_t)(tok0 + row) * p.nq + head) * D;
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                float part[32];
                tmem_ld32(my_o + c, part);
                if (row_ok) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        uint32_t ww[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const __nv_bfloat162 v = __floats2bfloat162_rn(part[i + 2 * q] * inv, part[i + 2 * q + 1] * inv);
                            ww[q] = *reinterpret_cast<const uint32_t*>(&v);
                        }
                        *reinterpret_cast<uint4*>(orow + c + i) = make_uint4(ww[0], ww[1], ww[2], ww[3]);
                    }
                }
            }
        }
      }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 13) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                     :: "r"(tmem_base), "r"((uint32_t)PF8_TMEM_COLS) : "memory");
    }
}

// What this kernel takes (a scale that is not positive goes to the general kernel).
extern "C" int acorn_attention_prefill_f8_supported(int nq, int nkv, int d, int P) {
    return nkv > 0 && nq % nkv == 0 && (d == 64 || d == 128) && P >= 8 && P <= 4096 && (P & (P - 1)) == 0;
}

template <int D>
static int launch_prefill_f8(PrefillF8Params pp, int64_t num_pages, int tokens, int64_t ctas, cudaStream_t stream) {
    using L = PrefillF8<D>;
    const F8AttnParams& p = pp.a;
    CUtensorMap mq, mk, mv;
    int rc = make_map(&mq, p.q, tokens, (int64_t)p.nq * D, p.q_stride, 64, PF8_BM);
    if (rc) return rc;
    rc = make_code_maps(&mk, &mv, p, num_pages, D, p.logP < 7 ? 1 << p.logP : PF8_BN, CU_TENSOR_MAP_SWIZZLE_NONE, &pp.joint, &pp.v_first);
    if (rc) return rc;
    static AcornPerDevice configured;
    if (!configured.seen()) {
        const cudaError_t e = cudaFuncSetAttribute(attention_prefill_f8_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
        if (e != cudaSuccess) return (int)e;
        configured.mark();
    }
    return acorn_launch(attention_prefill_f8_kernel<D>, dim3((unsigned)ctas), dim3(PF8_THREADS), L::SMEM, stream, mq, mk, mv, pp);
}

extern "C" int acorn_attention_prefill_f8(const void* q, int64_t q_stride, int tokens, void* out, const void* k_pages,
                                          const void* v_pages, const void* scales, int64_t num_pages, const int* block_table,
                                          const int* page_base, int table_stride, const int* row_start, const int* row_pos,
                                          const int* tiles, int n_tiles, int nq, int nkv, int d, int P, float scale, int window,
                                          int chunk, int keep, const float* sink, cudaStream_t stream) {
    if (n_tiles <= 0) return 0;
    if (!acorn_attention_prefill_f8_supported(nq, nkv, d, P) || q_stride % 8 != 0 || ((uintptr_t)q & 15) || !(scale > 0.f))
        return ACORN_ERR_UNSUPPORTED;
    PrefillF8Params pp;
    F8AttnParams& p = pp.a;
    p.q = (const bf16*)q; p.q_stride = q_stride; p.out = (bf16*)out; p.k_pages = (const uint8_t*)k_pages;
    p.v_pages = (const uint8_t*)v_pages; p.scales = (const uint8_t*)scales; p.block_table = block_table; p.page_base = page_base;
    p.row_start = row_start; p.row_pos = row_pos; p.tiles = tiles; p.sink = sink; p.table_stride = table_stride;
    p.nq = nq; p.nkv = nkv; p.mask = {window, chunk, keep}; p.scale_log2 = scale * 1.4426950408889634f;
    p.logP = acorn_log2_exact_tc(P);
    pp.pairs = (nq / nkv + 1) / 2;
    const int64_t ctas = (int64_t)n_tiles * nkv * pp.pairs;
    if (ctas > 0x7fffffff) return ACORN_ERR_UNSUPPORTED;
    return d == 128 ? launch_prefill_f8<128>(pp, num_pages, tokens, ctas, stream) : launch_prefill_f8<64>(pp, num_pages, tokens, ctas, stream);
}

extern "C" int acorn_attention_prefill_f8_error() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_attn_pre_f8_error, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_attn_pre_f8_error, &zero, sizeof(int));
    return v;
}

ACORN_ERROR_WORD_SETTER(acorn_attention_prefill_f8_set_error_word)
