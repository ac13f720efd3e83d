// Prefill attention over the pages of the 8-bit cache (f8_cache.cuh), head sizes 64 and 128: causal attention of tiles of 128
// consecutive queries of one request, on the 5th-generation tensor cores.
//
// Three kernels.
// 1. The keys and values of the rows that have tiles become bfloat16 rows, [kv head][place of the row + key], which is exact (code *
//    2^e is a bfloat16 number).  Done once a call, it reads and writes 5 bytes a number; turned into operand tiles by warps of the attention
//    kernel itself, every (tile, pair of heads) did it again, in competition with the softmax for the integer pipe and with the matrix
//    instructions for shared memory (8,192 tokens, 32 heads over 8: 840 us).
//    A row without tiles is left alone (2,048 tokens beside eight rows of 4,000 keys that decode: 98 us with theirs made too, 58 without).
//    Keys outside a row's range within its blocks of 128 get zero rows, so that whatever a slot of a page holds that was never
//    written, nothing of it is read; a row that is no number gets a NaN key, which spoils the queries that read it, and a zero value.
// 2. S = Q K^T and O += P V by tcgen05.mma with the accumulators in tensor memory.  One CTA per (tile, pair of query heads
//    that share a key/value head, split), one CTA to an SM.  The two heads ("units") read the same K and V tiles and take turns on
//    the tensor cores.
//      warps 0-7   softmax of unit 0, warps 8-15 of unit 1.  A query row (= TMEM lane) belongs to two threads, 64 keys of a
//                  block each: a block's scores pass through the softmax in half the time that one thread a row takes, and
//                  that time, not the tensor cores' or the exponentials', is what a unit's turn waits for.
//                  Weights are taken against a reference maximum that both threads of a row share; it moves when either of them
//                  saw a score beyond it by more than 2^24 (one vote of the unit's 256 threads a block; the first block is looked
//                  through for its maximum before anything else), and only then the two exchange their maxima, read the
//                  block again and scale O.  2^24: a weight keeps its 8 bits in bfloat16 whatever its size, and a move costs a unit
//                  half a block's time again (at 2^8 every third block of 8,192 tokens had one, 595 us; float32 sums of 2^17
//                  such weights overflow at values of 2^86).
//      warp 16     producer: Q (once), K and V tiles by TMA into a ring of five.
//      warp 17     MMA issuer (converged; one elected lane issues): per block j and unit u, O_u += P_u[j] V_j with P from
//                  tensor memory, then S_u = Q_u K_{j+1}^T into the columns P_u[j] was read from.
//    The softmax warps take 104 registers a thread, the fourth of a warpgroup's that the others leave them (twenty warps get
//    96 each; two are there for the split, which goes by warpgroups).
//    Tensor memory (512 columns): S / P of unit u at columns 128 u, O of unit u at 256 + 128 u.
// 3. Where the tiles are few, a tile's keys are split over several CTAs, whose results (float32, normalised, with the logarithm of
//    their sums) are joined by a third kernel.
//
// Every mbarrier wait is bounded; a wait that gives up records g_attn_pre_f8_error and the CTA drains: it ends, and its tensor
// memory is given back, when the copies and products that it issued are done.
#include "f8_tma.cuh"

#define PF8_BM 128
#define PF8_BN 128
#define PF8_SLOTS 5
#define PF8_THREADS 640
#define PF8_GROW_LOG2 24.0f
#define PF8_TMEM_COLS 512

__device__ int g_attn_pre_f8_error = 0;

struct PrefillF8Params {
    F8AttnParams a;
    int pairs;                // ceil((nq / nkv) / 2): CTAs per (tile, kv head, split)
    int n_tiles, rows;        // rows: of the block table
    const int* slot_rows;     // [slots]: the rows that have tiles, each once; or null: f8_place has the rule
    int slots;
    int cap;                  // without slot_rows: keys a slot has room for, a multiple of 128
    int room;                 // keys the scratch has room for, of one kv head
    int kvh0, kvhs;           // the kv heads of this pass
    int num_splits;
    bf16* k_rows;             // [kvhs, room, D]
    bf16* v_rows;
    float* part_o;            // [splits, n_tiles, 128, nq, D] where num_splits > 1
    float* part_lse;          // [splits, n_tiles, 128, nq]
};

// A row's blocks of 128 keys: those a rule's range covers, lo .. hi, with the kept first keys in front as blocks of their own.
struct F8Blocks {
    int lo, hi, nkb, n;
    __device__ __forceinline__ F8Blocks(const AttnMask& m, int pos0, int n_q) {
        hi = pos0 + n_q;                                             // keys < hi are read
        lo = mask_lo(m, pos0) & ~(PF8_BN - 1);                       // the first query's rule starts first
        nkb = (m.keep > 0 && lo > 0) ? min((m.keep + PF8_BN - 1) / PF8_BN, lo / PF8_BN) : 0;
        n = n_q > 0 ? nkb + (hi - lo + PF8_BN - 1) / PF8_BN : 0;
    }
    __device__ __forceinline__ int key0(int j) const { return j < nkb ? j * PF8_BN : lo + (j - nkb) * PF8_BN; }
};

// The key that a row's place starts with: the first whose page the row still holds, down to a multiple of 128.
__device__ __forceinline__ int f8_slot_key(const F8AttnParams& p, int r) { return (p.page_base[r] << p.logP) & ~(PF8_BN - 1); }

// Where in the scratch (in keys) a row's place starts; -1 for a row that has no tile.  The rows of a list lie one behind the other, each
// with as many blocks of 128 keys as it holds.  Without a list a place has room for the widest row of the table, and is that of the row's
// number, or where there are fewer tiles than rows that of the row's first tile.  `tiled`: the caller has the row from a tile.  All
// threads of a warp call it.
__device__ __forceinline__ int f8_place(const PrefillF8Params& pp, int r, bool tiled) {
    if (pp.slots == 1 && (tiled || pp.rows == 1 || pp.slot_rows != nullptr)) return 0;
    if (pp.slot_rows == nullptr && tiled && pp.n_tiles >= pp.rows) return r * pp.cap;
    const F8AttnParams& p = pp.a;
    const int lane = threadIdx.x & 31;
    if (pp.slot_rows != nullptr) {
        int before = 0;
        for (int s0 = 0; s0 < pp.slots; s0 += 32) {
            const int q = s0 + lane < pp.slots ? pp.slot_rows[s0 + lane] : -1;
            const int hi = q < 0 ? 0 : p.row_pos[q] + p.row_start[q + 1] - p.row_start[q];
            const int keys = q < 0 ? 0 : (hi + PF8_BN - 1) / PF8_BN * PF8_BN - f8_slot_key(p, q);
            const uint32_t hit = __ballot_sync(0xffffffffu, q == r);
            const int upto = hit ? __ffs(hit) - 1 : 32;
            before += __reduce_add_sync(0xffffffffu, lane < upto ? keys : 0);
            if (hit) return before;
        }
        return -1;
    }
    for (int t0 = 0; t0 < pp.n_tiles; t0 += 32) {
        const uint32_t hit = __ballot_sync(0xffffffffu, t0 + lane < pp.n_tiles && p.tiles[2 * min(t0 + lane, pp.n_tiles - 1)] == r);
        if (hit) return (pp.n_tiles >= pp.rows ? r : t0 + __ffs(hit) - 1) * pp.cap;
    }
    return -1;
}

// ---------------------------------------------------------------- 1. pages to rows of bfloat16

#define RB_THREADS 256

// A CTA takes a part of a block of 128 keys, 16 codes of a key and of its value a thread, of one kv head of the pass and one
// slot: a call of 2,048 tokens has some hundreds of CTAs then, whose chains of lookups overlap (a whole block a CTA: 10.9 us, 3 of
// them the bytes).
template <int D>
__global__ void __launch_bounds__(RB_THREADS) read_pages_f8_kernel(const PrefillF8Params pp) {
    const F8AttnParams& p = pp.a;
    pdl_wait();
    pdl_trigger();
    const int slot = blockIdx.z, kvh = pp.kvh0 + blockIdx.y;
    const int r = pp.rows == 1 ? 0 : pp.slot_rows != nullptr ? pp.slot_rows[slot] : pp.n_tiles < pp.rows ? p.tiles[2 * slot] : slot;
    int place = 0;
    if (pp.slot_rows == nullptr) {
        place = f8_place(pp, r, false);
        if (place != slot * pp.cap) return;                          // no tile reads the row, or another tile of the row came first
    }
    const F8Blocks b(p.mask, p.row_pos[r], p.row_start[r + 1] - p.row_start[r]);
    const int* table = p.block_table + (int64_t)r * p.table_stride - p.page_base[r];
    const int first_key = p.page_base[r] << p.logP, slot_key = f8_slot_key(p, r), pmask = (1 << p.logP) - 1;
    constexpr int PIECES = D / 16, KEYS = RB_THREADS / PIECES, PARTS = PF8_BN / KEYS;
    const int piece = threadIdx.x % PIECES;
    bool placed = pp.slot_rows == nullptr;
    for (int part = blockIdx.x; part < b.n * PARTS; part += gridDim.x) {
        const int key0 = b.key0(part / PARTS), key = key0 + part % PARTS * KEYS + threadIdx.x / PIECES;
        if (key0 < slot_key) continue;                               // (a kept block whose pages are gone)
        uint4 kc = make_uint4(0u, 0u, 0u, 0u), vc = kc;
        float ks = 0.f, vs = 0.f;
        if (key >= first_key && key < b.hi) {
            const int64_t at = (((int64_t)table[key >> p.logP] * p.nkv + kvh) << p.logP) + (key & pmask);
            kc = *reinterpret_cast<const uint4*>(p.k_pages + at * D + 16 * piece);
            vc = *reinterpret_cast<const uint4*>(p.v_pages + at * D + 16 * piece);
            const uint32_t bytes = *reinterpret_cast<const uint16_t*>(p.scales + 2 * at);
            ks = f8_scale(bytes & 255u);
            vs = f8_scale(bytes >> 8);
            if (isnan(ks) || isnan(vs)) { ks = __uint_as_float(0x7fc00000u); vs = 0.f; }
        }
        const uint32_t kw[4] = {kc.x, kc.y, kc.z, kc.w}, vw[4] = {vc.x, vc.y, vc.z, vc.w};
        uint32_t ko[8], vo[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const float2 a = f8_codes2(kw[q >> 1] >> (16 * (q & 1))), c = f8_codes2(vw[q >> 1] >> (16 * (q & 1)));
            const __nv_bfloat162 ab = __floats2bfloat162_rn(a.x * ks, a.y * ks), cb = __floats2bfloat162_rn(c.x * vs, c.y * vs);
            ko[q] = *reinterpret_cast<const uint32_t*>(&ab);
            vo[q] = *reinterpret_cast<const uint32_t*>(&cb);
        }
        if (!placed) {                                               // looked up while the first codes are on their way
            place = f8_place(pp, r, false);
            if (place + (b.hi + PF8_BN - 1) / PF8_BN * PF8_BN - slot_key > pp.room) {       // the caller's lengths were too short
                if (threadIdx.x == 0) tc_fail(&g_attn_pre_f8_error, 10, ACORN_KERNEL_ATTN_PREFILL_F8);
                return;
            }
            placed = true;
        }
        const int64_t out = ((int64_t)blockIdx.y * pp.room + place + (key - slot_key)) * D + 16 * piece;
        uint4* kd = reinterpret_cast<uint4*>(pp.k_rows + out);
        uint4* vd = reinterpret_cast<uint4*>(pp.v_rows + out);
        kd[0] = make_uint4(ko[0], ko[1], ko[2], ko[3]); kd[1] = make_uint4(ko[4], ko[5], ko[6], ko[7]);
        vd[0] = make_uint4(vo[0], vo[1], vo[2], vo[3]); vd[1] = make_uint4(vo[4], vo[5], vo[6], vo[7]);
    }
}

// ---------------------------------------------------------------- 2. attention

template <int D> struct PrefillF8 {
    static constexpr int HALVES = D / 64;
    static constexpr int HALF_BYTES = PF8_BN * 128;                  // [128 rows x 64 entries] bf16
    static constexpr int Q_BYTES = HALVES * PF8_BM * 128;            // one unit
    static constexpr int TILE_BYTES = HALVES * HALF_BYTES;           // a K or V tile
    static constexpr int TILES = 2 * Q_BYTES;                        // offsets in shared memory
    static constexpr int BARS = TILES + PF8_SLOTS * TILE_BYTES;
    // q_full, full, empty [SLOTS], s_full, p_full, o_done [unit], drained
    static constexpr int NUM_BARS = 1 + 2 * PF8_SLOTS + 6 + 1;
    static constexpr int SHARED = BARS + NUM_BARS * 8 + 16;          // [unit][half][row]: what the two threads of a row exchange
    static constexpr int SMEM = SHARED + 2 * 2 * PF8_BM * 4;
};

// Of columns c, those up to `last` are seen that are not before `first` or are before `keep` (all relative to the first one).
__device__ __forceinline__ void pf8_mask(float (&s)[32], int last, int first, int keep) {
#pragma unroll
    for (int c = 0; c < 32; ++c) s[c] = c <= last && (c >= first || c < keep) ? s[c] : -INFINITY;
}

__device__ __forceinline__ float pf8_max(const float (&s)[32], float m) {
    float a = m, b = -INFINITY;
#pragma unroll
    for (int c = 0; c < 32; c += 4) {
        a = fmaxf(a, fmaxf(s[c], s[c + 1]));
        b = fmaxf(b, fmaxf(s[c + 2], s[c + 3]));
    }
    return fmaxf(a, b);
}

// w[i] = bf16x2(2^(s[2i] * scale - m), 2^(s[2i+1] * scale - m)); returns the sum of the 32 values.
__device__ __forceinline__ float pf8_exp_pack(const float (&s)[32], float scale, float neg_m, uint32_t* w) {
    float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 32; c += 2) {
        const float a = fast_exp2(fmaf(s[c], scale, neg_m));
        const float b = fast_exp2(fmaf(s[c + 1], scale, neg_m));
        ps[(c >> 1) & 3] += a + b;
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        w[c >> 1] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return (ps[0] + ps[1]) + (ps[2] + ps[3]);
}

// The scale with which a row whose reference is m (in units of log2, at the softmax's scale) is exponentiated.  A weight's
// exponent is one rounding of s * scale - m, so that the rounding of m itself is a factor that all weights of the row share;
// beyond 2^29 it could be one that overflows.  There neighbouring float32 scores differ by 32 or more, so that all weights but those
// of the largest score vanish, and they still do at a scale that brings m to 2^29.
__device__ __forceinline__ float pf8_row_scale(float scale_log2, float m) {
    const int beyond = (int)(__float_as_uint(m) >> 23 & 255u) - 127 - 29;
    return beyond > 0 ? scale_log2 * f8_pow2(-beyond) : scale_log2;
}

// Meets the 256 threads of a unit; whether `v` holds for any of them.
__device__ __forceinline__ bool unit_any(int unit, bool v) {
    uint32_t r;
    tc_fence_before();
    asm volatile("{\n .reg .pred a, b;\n setp.ne.u32 a, %1, 0;\n barrier.cta.red.or.pred b, %2, 256, a;\n selp.u32 %0, 1, 0, b;\n}\n"
                 : "=r"(r) : "r"((uint32_t)v), "r"(unit + 1) : "memory");
    tc_fence_after();
    return r != 0;
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
    const uint32_t full0 = q_full + 8, empty0 = full0 + 8 * PF8_SLOTS;
    const uint32_t s_full0 = empty0 + 8 * PF8_SLOTS, p_full0 = s_full0 + 16, o_done0 = p_full0 + 16, drained = o_done0 + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::NUM_BARS);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // CTAs are started in the order of the tile list; CTAs next to one another share a tile and mostly a key/value head.
    const int per_tile = pp.kvhs * pp.pairs;
    const int tile = (int)(blockIdx.x / per_tile), split = blockIdx.y;
    const int kvp = (int)(blockIdx.x % per_tile) / pp.pairs, pair = (int)(blockIdx.x % per_tile) % pp.pairs;
    const int rep = p.nq / p.nkv;
    const int head0 = (pp.kvh0 + kvp) * rep + 2 * pair;
    const int units = (2 * pair + 1 < rep) ? 2 : 1;
    if (tc_smem(smem) & 1023u) {            // the swizzled tiles need a 1024-byte aligned base
        if (threadIdx.x == 0) tc_fail(&g_attn_pre_f8_error, 9, ACORN_KERNEL_ATTN_PREFILL_F8);
        return;
    }
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(drained, 1);
        for (int s = 0; s < PF8_SLOTS; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int u = 0; u < 2; ++u) { mbar_init(s_full0 + 8 * u, 1); mbar_init(p_full0 + 8 * u, 8); mbar_init(o_done0 + 8 * u, 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 17) {
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
    const F8Blocks blocks(p.mask, pos0, n_q);
    const int per = (blocks.n + pp.num_splits - 1) / pp.num_splits;
    const int j0 = min(blocks.n, split * per), nb = min(blocks.n, j0 + per) - j0;        // this split's blocks

    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 16) {
            // ------------------------------------------------------------ producer
            const int first = f8_slot_key(p, r), place = f8_place(pp, r, true);
            const int row0 = kvp * pp.room + max(place, 0) - first;
            if (nb > 0 && elect_one()) {
                mbar_expect_tx(q_full, units * L::Q_BYTES);
                for (int u = 0; u < units; ++u)
                    for (int h = 0; h < L::HALVES; ++h)
                        tma_load_2d(tc_smem(smem) + u * L::Q_BYTES + h * PF8_BM * 128, &map_q, q_full, (head0 + u) * D + 64 * h, tok0);
            }
            int slot = 0, phase = 0, n = 0;
            for (; n < 2 * nb; ++n) {                                    // K_0 V_0 K_1 V_1 ...
                const bool got = mbar_wait(empty0 + 8 * slot, phase ^ 1);
                if (!got && lane == 0) tc_fail(&g_attn_pre_f8_error, 1, ACORN_KERNEL_ATTN_PREFILL_F8);
                if (!__all_sync(0xffffffffu, got)) break;
                const CUtensorMap* map = n & 1 ? &map_v : &map_k;
                const int y = row0 + max(blocks.key0(j0 + (n >> 1)), first);
                if (elect_one()) {
                    mbar_expect_tx(full0 + 8 * slot, L::TILE_BYTES);
                    for (int h = 0; h < L::HALVES; ++h)
                        tma_load_2d(tc_smem(smem + L::TILES) + slot * L::TILE_BYTES + h * L::HALF_BYTES, map, full0 + 8 * slot, 64 * h, y);
                }
                if (++slot == PF8_SLOTS) { slot = 0; phase ^= 1; }
            }
            if ((place < 0 || (pp.slot_rows != nullptr && pp.slots == 1 && pp.slot_rows[0] != r)) && lane == 0)
                tc_fail(&g_attn_pre_f8_error, 11, ACORN_KERNEL_ATTN_PREFILL_F8);                           // a row that was not listed
            // all copies have landed before the CTA ends, also where the others gave up and read none of them
            if (nb > 0) mbar_wait(q_full, 0);
            for (int k = max(0, n - PF8_SLOTS); k < n; ++k) mbar_wait(full0 + 8 * (k % PF8_SLOTS), (k / PF8_SLOTS) & 1);
        } else if (warp == 17) {
            // ------------------------------------------------------------ MMA issuer
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
            auto issue_qk = [&](int u, int slot) {                      // S_u = Q_u K^T, K in `slot`
                const uint32_t klo = klo0 + slot * (L::TILE_BYTES >> 4);
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    umma_bf16_elect(tmem_s + u * 128, qlo + ((u * L::Q_BYTES + (k >> 2) * PF8_BM * 128) >> 4) + 2 * (k & 3),
                                    klo + (((k >> 2) * L::HALF_BYTES) >> 4) + 2 * (k & 3), IDESC_QK, k > 0 ? 1u : 0u);
                umma_commit_elect(s_full0 + 8 * u);
            };
            bool good = nb > 0 && wait_all(q_full, 0, 2) && wait_all(full0, 0, 3);
            int slot = 0, phase = 0;                                     // the next tile of the ring
            const bool issued = good;
            if (good) {
                for (int u = 0; u < units; ++u) issue_qk(u, 0);
                umma_commit_elect(empty0);
                slot = 1;
            }
            for (int j = 0; j < nb && good; ++j) {
                const int sv = slot, pv = phase;                         // V_j
                if (++slot == PF8_SLOTS) { slot = 0; phase ^= 1; }
                const int sk = slot, pk = phase;                         // K_{j+1}
                const bool has_next = j + 1 < nb;
                if (has_next) { if (++slot == PF8_SLOTS) { slot = 0; phase ^= 1; } }
                good = wait_all(full0 + 8 * sv, pv, 3);
                if (good && has_next) good = wait_all(full0 + 8 * sk, pk, 3);
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
                    // the next scores go where P was: the pipe runs them after the product above
                    if (has_next) issue_qk(u, sk);
                    else umma_commit_elect(o_done0 + 8 * u);
                }
                if (!good) break;
                umma_commit_elect(empty0 + 8 * sv);
                if (has_next) umma_commit_elect(empty0 + 8 * sk);
            }
            // the products are done before the tensor memory is given back, also where somebody gave up in between
            if (issued) {
                umma_commit_elect(drained);
                mbar_wait(drained, 0);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        const int u = warp >> 3, half = (warp >> 2) & 1;
        if (u < units) {
            // ------------------------------------------------------------ softmax and output
            const int row = (warp & 3) * 32 + lane;                      // query row = TMEM lane
            const int head = head0 + u;
            const bool row_ok = row < n_q;
            const int last_seen = row_ok ? pos0 + row : -1, first_seen = mask_lo(p.mask, pos0 + row);
            const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t unit_s = tmem_s + lane_addr + u * 128, my_s = unit_s + 64 * half, my_p = unit_s + 32 * half;
            const uint32_t my_o = tmem_o + lane_addr + u * 128 + half * (D / 2);
            const uint32_t s_full = s_full0 + 8 * u, p_full = p_full0 + 8 * u, o_done = o_done0 + 8 * u;
            float* mine = reinterpret_cast<float*>(smem + L::SHARED) + (2 * u + half) * PF8_BM + row;
            float* other = reinterpret_cast<float*>(smem + L::SHARED) + (2 * u + 1 - half) * PF8_BM + row;
            const int last_lo = n_q > 0 ? mask_lo(p.mask, blocks.hi - 1) : 0;            // the last query's rule starts last
            float m_ref = -INFINITY, l_run = 0.f;                        // the reference in units of log2
            float scale = p.scale_log2, neg_m = 0.f;                     // what the row's scores are exponentiated with
            bool good = nb > 0;
            auto refer = [&](float top) {                                // to the larger of the two threads' maxima
                m_ref = top * p.scale_log2;                              // the scale is positive
                scale = pf8_row_scale(p.scale_log2, m_ref);
                neg_m = -(top * scale);
            };
            if (good) {
                const bool got = mbar_wait(s_full, 0);
                if (!got) tc_fail(&g_attn_pre_f8_error, 5, ACORN_KERNEL_ATTN_PREFILL_F8);
                tc_fence_after();
                const int block0 = blocks.key0(j0), key0 = block0 + 64 * half;
                float s[32], top = -INFINITY;
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    tmem_ld32(my_s + 32 * h, s);
                    pf8_mask(s, last_seen - key0 - 32 * h, first_seen - key0 - 32 * h, p.mask.keep - key0 - 32 * h);
                    top = pf8_max(s, top);
                }
                *mine = top;
                good = !unit_any(u, !got);                               // (a wait that gave up makes the whole unit stop)
                top = fmaxf(top, *other);
                if (top > -INFINITY) refer(top);
            }
            for (int j = 0; j < nb && good; ++j) {
                // S of block j is complete; so is P V of block j-1, issued before it: O is stable
                bool got = mbar_wait(s_full, j & 1);
                if (!got) tc_fail(&g_attn_pre_f8_error, 6, ACORN_KERNEL_ATTN_PREFILL_F8);
                tc_fence_after();
                const int block0 = blocks.key0(j0 + j), key0 = block0 + 64 * half;
                // a block that every query of the tile sees whole needs no mask
                const bool masked = block0 + PF8_BN - 1 > pos0 || block0 < last_lo || n_q < PF8_BM;
                float s[32];
                uint32_t w[32];
                float top = -INFINITY, psum = 0.f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    tmem_ld32(my_s + 32 * h, s);
                    if (masked) pf8_mask(s, last_seen - key0 - 32 * h, first_seen - key0 - 32 * h, p.mask.keep - key0 - 32 * h);
                    top = pf8_max(s, top);
                    psum += pf8_exp_pack(s, scale, neg_m, w + 16 * h);
                }
                const float mx = top * p.scale_log2;                     // the scale is positive
                if (unit_any(u, !got || mx > m_ref + PF8_GROW_LOG2)) {
                    *mine = top;
                    good = !unit_any(u, !got);
                    if (!good) break;
                    const float both = fmaxf(top, *other), mb = both * p.scale_log2;
                    float corr = 1.f;
                    if (mb > m_ref + PF8_GROW_LOG2) {
                        corr = fast_exp2(m_ref - mb);                    // m_ref = -inf: 0
                        l_run *= corr;
                        refer(both);
                    }
                    psum = 0.f;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        tmem_ld32(my_s + 32 * h, s);
                        if (masked) pf8_mask(s, last_seen - key0 - 32 * h, first_seen - key0 - 32 * h, p.mask.keep - key0 - 32 * h);
                        psum += pf8_exp_pack(s, scale, neg_m, w + 16 * h);
                    }
                    if (j > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll 1
                        for (int c = 0; c < D / 2; c += 32) {
                            tmem_ld32(my_o + c, s);
#pragma unroll
                            for (int i = 0; i < 32; ++i) s[i] *= corr;
                            tmem_st32(my_o + c, s);
                        }
                    }
                    unit_any(u, false);                                  // nobody reads S any more: P may be written over it
                }
                l_run += psum;
                tmem_st32_raw(my_p, w);                                  // column c of P holds keys 2c and 2c + 1
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full);
            }
            if (good) {
                const bool got = mbar_wait(o_done, 0);
                if (!got) tc_fail(&g_attn_pre_f8_error, 8, ACORN_KERNEL_ATTN_PREFILL_F8);
                unit_any(u, false);                                      // (the last exchange's values have been read)
                *mine = l_run;
                unit_any(u, false);
                good = __all_sync(0xffffffffu, got);
            }
            if (good) {
                tc_fence_after();
                float total = l_run + *other;
                // a sink is one more term of the denominator, in the first split; the denominator is taken against the larger of the
                // reference and the sink, so that neither overflows
                const float sink = p.sink && row_ok && split == 0 ? p.sink[head] * 1.4426950408889634f : -INFINITY;
                // (a split that holds no key of the row: the sink alone; NaN keys leave no maximum, but a NaN sum)
                const bool empty = m_ref == -INFINITY && total == 0.f;
                float against = m_ref, shrink = 1.f;
                if (sink != -INFINITY && !empty) {
                    against = fmaxf(m_ref, sink);
                    shrink = exp2f(m_ref - against);
                    total = total * shrink + exp2f(sink - against);
                }
                const float inv = row_ok ? shrink / total : 0.f;
                const int64_t out_row = (int64_t)(tok0 + row) * p.nq + head;
                const int64_t part_row = (((int64_t)split * pp.n_tiles + tile) * PF8_BM + row) * p.nq + head;
                if (pp.num_splits > 1 && row_ok && half == 0) pp.part_lse[part_row] = empty ? sink : against + log2f(total);
#pragma unroll 1
                for (int c = 0; c < D / 2; c += 32) {
                    float part[32];
                    tmem_ld32(my_o + c, part);
                    if (!row_ok) continue;
                    if (pp.num_splits > 1) {
                        float4* dst = reinterpret_cast<float4*>(pp.part_o + part_row * D + half * (D / 2) + c);
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            dst[i >> 2] = empty ? make_float4(0.f, 0.f, 0.f, 0.f)
                                                : make_float4(part[i] * inv, part[i + 1] * inv, part[i + 2] * inv, part[i + 3] * inv);
                        continue;
                    }
                    uint4* dst = reinterpret_cast<uint4*>(p.out + out_row * D + half * (D / 2) + c);
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        uint32_t ww[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const __nv_bfloat162 v = __floats2bfloat162_rn(part[i + 2 * q] * inv, part[i + 2 * q + 1] * inv);
                            ww[q] = *reinterpret_cast<const uint32_t*>(&v);
                        }
                        dst[i >> 3] = make_uint4(ww[0], ww[1], ww[2], ww[3]);
                    }
                }
            } else if (nb == 0 && pp.num_splits > 1 && row_ok && half == 0) {
                // no blocks for this split (never the first): no weight in the join, its outputs are not read
                pp.part_lse[(((int64_t)split * pp.n_tiles + tile) * PF8_BM + row) * p.nq + head] = -INFINITY;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 17) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                     :: "r"(tmem_base), "r"((uint32_t)PF8_TMEM_COLS) : "memory");
    }
}

// ---------------------------------------------------------------- 3. the splits joined

// One warp per (query of a tile, head of the pass); 4 entries a lane (2 at head size 64).
template <int D>
__global__ void __launch_bounds__(256) attention_prefill_f8_join_kernel(const PrefillF8Params pp) {
    constexpr int E = D / 32;
    pdl_wait();
    pdl_trigger();
    const F8AttnParams& p = pp.a;
    const int rep = p.nq / p.nkv, heads = pp.kvhs * rep;
    const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (item >= (int64_t)pp.n_tiles * PF8_BM * heads) return;
    const int head = pp.kvh0 * rep + (int)(item % heads), row = (int)(item / heads % PF8_BM), tile = (int)(item / heads / PF8_BM);
    const int r = p.tiles[2 * tile], tok = p.row_start[r] + p.tiles[2 * tile + 1] + row;
    if (tok >= p.row_start[r + 1]) return;
    const int64_t step = (int64_t)pp.n_tiles * PF8_BM * p.nq, at0 = ((int64_t)tile * PF8_BM + row) * p.nq + head;
    float top = -INFINITY;
    for (int s = 0; s < pp.num_splits; ++s) top = fmaxf(top, pp.part_lse[at0 + s * step]);
    float sum = 0.f, acc[E];
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = 0.f;
    for (int s = 0; s < pp.num_splits; ++s) {
        const float lse = pp.part_lse[at0 + s * step];
        if (lse == -INFINITY) continue;
        const float f = exp2f(lse - top);
        sum += f;
        const float* o = pp.part_o + (at0 + s * step) * D + lane * E;
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] = fmaf(f, o[i], acc[i]);
    }
    bf16* dst = p.out + ((int64_t)tok * p.nq + head) * D + lane * E;
    const float inv = 1.f / sum;
#pragma unroll
    for (int i = 0; i < E; i += 2) *reinterpret_cast<__nv_bfloat162*>(dst + i) = __floats2bfloat162_rn(acc[i] * inv, acc[i + 1] * inv);
}

// ---------------------------------------------------------------- host

// What these kernels take (a scale that is not positive goes to the general kernel).
extern "C" int acorn_attention_prefill_f8_supported(int nq, int nkv, int d, int P) {
    return nkv > 0 && nq % nkv == 0 && (d == 64 || d == 128) && P >= 1 && P <= 4096 && (P & (P - 1)) == 0;
}

template <int D>
static int launch_prefill_f8(const PrefillF8Params& pp, int tokens, int blocks, cudaStream_t stream) {
    using L = PrefillF8<D>;
    const F8AttnParams& p = pp.a;
    CUtensorMap mq, mk, mv;
    const int64_t rows = (int64_t)pp.kvhs * pp.room;
    if (rows > 0x7fffffff) return ACORN_ERR_UNSUPPORTED;
    int rc = make_map(&mq, p.q, tokens, (int64_t)p.nq * D, p.q_stride, 64, PF8_BM);
    if (rc) return rc;
    rc = make_map(&mk, pp.k_rows, rows, D, D, 64, PF8_BN);
    if (rc) return rc;
    rc = make_map(&mv, pp.v_rows, rows, D, D, 64, PF8_BN);
    if (rc) return rc;
    static AcornPerDevice configured;
    if (!configured.seen()) {
        const cudaError_t e = cudaFuncSetAttribute(attention_prefill_f8_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
        if (e != cudaSuccess) return (int)e;
        configured.mark();
    }
    rc = acorn_launch(read_pages_f8_kernel<D>, dim3(blocks, pp.kvhs, pp.slots), dim3(RB_THREADS), 0, stream, pp);
    if (rc) return rc;
    const int64_t ctas = (int64_t)pp.n_tiles * pp.kvhs * pp.pairs;
    rc = acorn_launch(attention_prefill_f8_kernel<D>, dim3((unsigned)ctas, pp.num_splits), dim3(PF8_THREADS), L::SMEM, stream, mq, mk, mv, pp);
    if (rc || pp.num_splits == 1) return rc;
    const int64_t items = (int64_t)pp.n_tiles * PF8_BM * pp.kvhs * (p.nq / p.nkv);
    return acorn_launch(attention_prefill_f8_join_kernel<D>, dim3((unsigned)((items + 7) / 8)), dim3(256), 0, stream, pp);
}

// slot_rows [slots]: the rows that have tiles, each once, or null with `slots` = min(rows of the table, tiles) of `cap` keys each;
// k_rows / v_rows: [kvhs, room, d] bfloat16 for the kv heads kvh0 .. kvh0 + kvhs - 1 of this pass; blocks: CTAs along a row's keys.
extern "C" int acorn_attention_prefill_f8(const void* q, int64_t q_stride, int tokens, void* out, const void* k_pages,
                                          const void* v_pages, const void* scales, const int* block_table, const int* page_base,
                                          int table_stride, int rows, const int* row_start, const int* row_pos, const int* tiles,
                                          int n_tiles, int nq, int nkv, int d, int P, float scale, int window, int chunk, int keep,
                                          const float* sink, int kvh0, int kvhs, void* k_rows, void* v_rows, const int* slot_rows,
                                          int slots, int cap, int room, int blocks, int num_splits, float* part_o, float* part_lse, cudaStream_t stream) {
    if (n_tiles <= 0) return 0;
    if (!acorn_attention_prefill_f8_supported(nq, nkv, d, P) || q_stride % 8 != 0 || ((uintptr_t)q & 15) || !(scale > 0.f) ||
        cap % PF8_BN || room % PF8_BN || room < 1 || slots < 1 || slots > 65535 || kvhs < 1 || kvhs > 65535 || kvh0 < 0 || kvh0 + kvhs > nkv || blocks < 1 ||
        num_splits < 1 || num_splits > 65535 || (num_splits > 1 && (part_o == nullptr || part_lse == nullptr)) ||
        (slot_rows == nullptr && (slots != (n_tiles < rows ? n_tiles : rows) || (int64_t)slots * cap > room)))
        return ACORN_ERR_UNSUPPORTED;
    PrefillF8Params pp;
    F8AttnParams& p = pp.a;
    p.q = (const bf16*)q; p.q_stride = q_stride; p.out = (bf16*)out; p.k_pages = (const uint8_t*)k_pages;
    p.v_pages = (const uint8_t*)v_pages; p.scales = (const uint8_t*)scales; p.block_table = block_table; p.page_base = page_base;
    p.row_start = row_start; p.row_pos = row_pos; p.tiles = tiles; p.sink = sink; p.table_stride = table_stride;
    p.nq = nq; p.nkv = nkv; p.mask = {window, chunk, keep}; p.scale_log2 = scale * 1.4426950408889634f;
    p.logP = acorn_log2_exact_tc(P);
    pp.pairs = (nq / nkv + 1) / 2; pp.n_tiles = n_tiles; pp.rows = rows; pp.cap = cap; pp.room = room; pp.slot_rows = slot_rows; pp.slots = slots; pp.kvh0 = kvh0; pp.kvhs = kvhs;
    pp.num_splits = num_splits; pp.k_rows = (bf16*)k_rows; pp.v_rows = (bf16*)v_rows; pp.part_o = part_o; pp.part_lse = part_lse;
    if ((int64_t)n_tiles * kvhs * pp.pairs > 0x7fffffff || (int64_t)n_tiles * PF8_BM * nq > ((int64_t)1 << 33)) return ACORN_ERR_UNSUPPORTED;
    return d == 128 ? launch_prefill_f8<128>(pp, tokens, blocks, stream) : launch_prefill_f8<64>(pp, tokens, blocks, stream);
}

extern "C" int acorn_attention_prefill_f8_error() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_attn_pre_f8_error, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_attn_pre_f8_error, &zero, sizeof(int));
    return v;
}

ACORN_ERROR_WORD_SETTER(acorn_attention_prefill_f8_set_error_word)
