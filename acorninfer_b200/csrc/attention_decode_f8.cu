// Attention of few tokens a row over the pages of the 8-bit cache (f8_cache.cuh), head sizes 64 and 128: split-K flash decoding.
//
// A tile is up to 16 / rep tokens of one row (rep = nq / nkv query heads share a kv head);
// its (token, head) pairs are its query rows, so the tokens of a tile read their row's pages together.
// A producer warp brings the codes by TMA (swizzled; a box is the keys and the values of one page and head, through a map whose
// third dimension is the distance between the two page tensors) and their exponents by asynchronous copies into a ring of
// stages of 64 keys: an issued copy costs the warp some 130 clocks, which is what bounds a CTA at small pages.  Each of the four
// other warps takes 16 keys of a stage through m16n8k16 products whose sixteen rows are the keys (then the entries of the values) and
// whose eight columns are query rows; more than eight query rows are NH = 2 products on the same operands:
//   S' = K Q'   codes become half-precision numbers by one conversion a pair (e4m3 is exact in it); the queries are
//               brought to half precision by a power of two per row (their largest entry to 2^14 .. 2^15, so that a bfloat16
//               entry is exact unless it is 2^-28 of the largest), and both powers of two meet the score in float32.
//   P = 2^(t + e_v - m)   t the score in units of log2, e_v the exponent of the key's value row, m a reference near the largest
//               t + e_v so far: the value's power of two rides in the exponent, so that a weight is at most 2^14 (the reference
//               moves when it is outgrown by more) in half precision, with 11 bits where bfloat16 would keep 8, whatever the
//               sizes of the value rows.  Against the reference the common step needs no maximum across lanes, only a vote.
//   O' += V' P' on value codes as half-precision numbers (a weight's transpose within the warp is one movmatrix);
//   L += 2^(t - r)  the denominator in float32, r a reference near the largest t alone: m lies up to 120 to either side of the
//               scores (a row of zeros has e_v = -120), and 2^(t - m) summed would be infinite after 256 such keys.  The result is
//               O' / L 2^(m - r).
// The layouts of the fragments are chosen so that a lane's codes are whole 16-byte pieces of rows: the order of the head's
// entries in a product over them is free (Q is laid out the same way), and so is the order of the output's rows.
// Codes of keys that no query of the tile reads are replaced by zeros (a slot that was never written may hold anything).
//
// Which keys a CTA takes:
//   splits         one (tile, kv head, split) a CTA; the splits of a (tile, kv head), 2 to 8 or 16, are a thread-block cluster
//                  that joins them through distributed shared memory: one launch, for calls of little work;
//   even shares    as many CTAs as the device holds at once share all the chunks of 64 keys of all (tile, kv head) pairs out evenly,
//                  in order, so that a CTA walks from pair to pair: nobody waits for the longest row or for a last wave of few CTAs, and
//                  the codes of the next pair are on their way while the warps finish one (a CTA's start and end cost some 5
//                  us).  A pair that several CTAs had parts of is joined by a second, small kernel (some 4 us).  64 rows of 4,096
//                  keys of 8 kv heads of 128: 122 us whole, 111 in 3 splits, 97 in shares, 545 MB at 5.6 TB/s.
// What bounds it: memory where there is enough of it (that case's main kernel moves its bytes at 0.85 of the copy rate), else
// a warp's chain of some 300 instructions a chunk, 0.6 us (0.8 with the copies of pages of 16), and the start and the end.  The
// denominator's own reference costs up to 2.5 % at eight query rows and 1.5 to 6 at sixteen; warps that take whole rows of the join, rather
// than threads its entries, and move them as vectors, brought up to 7 % (8 rows of 4,000 keys 17.5, 17.8 with the reference, 16.6).
// Tried and taken back: the next chunk's scores formed among this one's weights (44 bytes spilled; 10 to 15 % slower at head size
// 128), four CTAs an SM at 96 registers (20 % slower a chunk), more than 16 splits through scratch (59 us for one row of 131,072
// keys in 48, as the shares).
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "f8_tma.cuh"
#include "mma_helpers.cuh"

namespace cg = cooperative_groups;

#define DF8_WARPS 4                         // compute warps; one more brings the codes
#define DF8_THREADS (32 * DF8_WARPS + 32)
#define DF8_CHUNK (16 * DF8_WARPS)
#define DF8_CLUSTER_MAX 16
#define DF8_GROW_LOG2 14.f                  // the reference maximum moves when a row's maximum outgrew it by more than this
                                            // (half-precision weights end at 2^16)
#define DF8_SUM_LOG2 64.f                           // and the denominator's by more than this (float32: room for 2^63 keys)
#define DF8_NONE (-3.402823466e38f)                 // a reference that no score has moved: every finite one is at least as large, and
                                                    // -infinity less it is -infinity, a weight of 0

__device__ int g_attn_dec_f8_error = 0;

#define DF8_SHARE_TILES 256                 // tiles that a CTA keeps the sizes of for the even shares
#define DF8_SHARE_MIN 4                     // chunks that a share has at least

struct DecodeF8Params {
    F8AttnParams a;
    int n_tiles, tile_tokens, num_splits;           // tile_tokens: the most tokens a tile holds; num_splits 0: even shares
    int joint, v_first;       // one box brings keys and values (the tensor at the lower address first), else two do
    // even shares: what the join needs
    float* part_o;            // [CTAs, 2, 8 NH, D]: the part that a CTA's share begins with, and the one that it ends with
    float* part_lse;          // [CTAs, 2, 8 NH]
    int4* plan;               // [n_tiles + 1]: chunks of the tiles before (of one kv head), chunks, first token, tokens; the last: chunks a share
};

template <int D, int NH> struct DecodeF8 {
    static constexpr int ROWS = 8 * NH;
    static constexpr int STAGES = D == 128 ? 3 : 6;
    static constexpr int ROWS_BYTES = DF8_CHUNK * D;                  // the codes of a stage's keys (or values)
    static constexpr int STAGE_BYTES = 2 * ROWS_BYTES;
    static constexpr int SCALE_BYTES = 2 * DF8_CHUNK;
    static constexpr int RECV_ROW = D + 4;                            // floats a received partial row takes: the output, then its log-sum
    static constexpr int RING = STAGES * STAGE_BYTES;
    static constexpr int MERGE_BYTES = DF8_WARPS * ROWS * (3 + D) * 4;
    static constexpr int MERGE = RING;                                // offsets in shared memory
    static constexpr int BARS = MERGE + MERGE_BYTES;
    static constexpr int SCALES = BARS + 2 * STAGES * 8;
    static constexpr int RECV = SCALES + STAGES * SCALE_BYTES;        // received rows of a cluster, or the sizes of the tiles
    static constexpr int SHARES = (DF8_SHARE_TILES + 4) * 4 + DF8_SHARE_TILES * 16;       // chunks before a tile; row, first token, tokens, position
    static_assert(RECV % 16 == 0 && MERGE % 16 == 0 && RECV_ROW % 4 == 0, "float4 and int4 accesses");
    // byte offset of the 16-byte piece `seg` of row `row` of a stage (boxes of 2^log_box keys, then as many values), as the
    // TMA's swizzle places it
    static __device__ __forceinline__ uint32_t at(int row, int seg) {
        return D == 128 ? (uint32_t)(row * 128 + ((seg ^ (row & 7)) << 4)) : (uint32_t)(row * 64 + ((seg ^ ((row >> 1) & 3)) << 4));
    }
};

// (not volatile: the compiler may move it among the conversions that feed it; two products on different sums are independent)
__device__ __forceinline__ void mma_f16_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// An 8 x 8 matrix of 16-bit elements across the warp (lane (g, i): row g, columns 2 i and 2 i + 1), transposed.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// max / sum over the eight lanes that share lane % 4
__device__ __forceinline__ float column_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 4);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

// Two or four neighbouring floats, moved together.
template <int E> struct alignas(4 * E) F8Floats { float v[E]; };
template <int E> __device__ __forceinline__ void st_cluster(uint32_t addr, const F8Floats<E>& x) {
    if constexpr (E == 4)
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" :: "r"(addr), "f"(x.v[0]), "f"(x.v[1]), "f"(x.v[2]), "f"(x.v[3]) : "memory");
    else
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" :: "r"(addr), "f"(x.v[0]), "f"(x.v[1]) : "memory");
}

// What a CTA needs to know of a tile.
struct F8Tile {
    int r, tok0, n_q, pos0, hi, lo, base_key, nkb, n_chunks;
    __device__ __forceinline__ F8Tile(const DecodeF8Params& dp, int ti) {
        const F8AttnParams& p = dp.a;
        r = p.tiles[2 * ti];
        const int q0 = p.tiles[2 * ti + 1];
        tok0 = p.row_start[r] + q0;
        n_q = max(0, min(dp.tile_tokens, p.row_start[r + 1] - tok0));
        pos0 = p.row_pos[r] + q0;
        keys(p);
    }
    __device__ __forceinline__ F8Tile(const F8AttnParams& p, const int4& v) : r(v.x), tok0(v.y), n_q(v.z), pos0(v.w) { keys(p); }
    __device__ __forceinline__ void keys(const F8AttnParams& p) {
        hi = pos0 + n_q;                                          // keys < hi are read by the tile
        lo = mask_lo(p.mask, pos0);                               // the first query's rule starts first
        base_key = lo & ~(DF8_CHUNK - 1);                         // chunks start at multiples of 64 keys
        // the kept first keys, where the rule's range starts beyond them, are chunks of their own in front
        nkb = (p.mask.keep > 0 && base_key > 0) ? min((p.mask.keep + DF8_CHUNK - 1) / DF8_CHUNK, base_key / DF8_CHUNK) : 0;
        n_chunks = n_q > 0 ? nkb + (hi - base_key + DF8_CHUNK - 1) / DF8_CHUNK : 0;
    }
    __device__ __forceinline__ int key0(int c) const { return c < nkb ? c * DF8_CHUNK : base_key + (c - nkb) * DF8_CHUNK; }
};

// The parts of (tile, kv head) pairs that a CTA takes, one after the other.
struct F8Walk {
    const int* before;        // even shares: chunks of the tiles before each, and the tiles (shared memory)
    const int4* tiles;
    int n_tiles, nkv, ti, kvh, c0, c1;
    int64_t at, end;          // of the share, in chunks of all pairs
    // even shares: units are ordered by tile, then kv head, then chunk
    __device__ __forceinline__ bool next() {
        if (at >= end) return false;
        int a = 0, b = n_tiles;                                   // the last tile that starts at or before `at`
        while (b - a > 1) {
            const int m = (a + b) >> 1;
            if ((int64_t)before[m] * nkv <= at) a = m; else b = m;
        }
        ti = a;
        const int n = before[a + 1] - before[a];                  // > 0: tiles without chunks start where the next one does
        const int64_t in = at - (int64_t)before[a] * nkv;
        kvh = (int)(in / n);
        c0 = (int)(in - (int64_t)kvh * n);
        c1 = (int)min((int64_t)n, c0 + (end - at));
        at += c1 - c0;
        return true;
    }
};

// Meets the compute warps; whether `v` holds for all of them.
__device__ __forceinline__ bool compute_all(bool v) {
    uint32_t r;
    asm volatile("{\n .reg .pred a, b;\n setp.ne.u32 a, %1, 0;\n barrier.cta.red.and.pred b, 1, %2, a;\n selp.u32 %0, 1, 0, b;\n}\n"
                 : "=r"(r) : "r"((uint32_t)v), "n"(32 * DF8_WARPS) : "memory");
    return r != 0;
}

// CTAs an SM: three, but two where sixteen rows of 128 entries need more than 128 registers a thread.  (Sixteen rows of 64, three
// against two, measured before the denominator had a reference of its own: 24 rows of 3 new tokens over a window of 1,024 19.1 us against
// 20.7, 41 of 2 over up to 1,700 22.9 against 28.0, 64 over 4,096 at sixteen heads a group 62.8 against 68.1.)
template <int D, int NH, bool SHARES>
__global__ void __launch_bounds__(DF8_THREADS, NH == 1 || D == 64 ? 3 : 2) attention_decode_f8_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                         const __grid_constant__ CUtensorMap map_v,
                                                                         const DecodeF8Params dp) {
    using L = DecodeF8<D, NH>;
    constexpr int ROWS = L::ROWS;
    constexpr int WORDS = D / 16;                              // 32-bit words of codes a lane holds of a key row; k-steps of a product;
                                                               // row tiles of the output
    extern __shared__ __align__(1024) uint8_t smem[];
    const F8AttnParams& p = dp.a;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
    const uint32_t full0 = tc_smem(bars), empty0 = tc_smem(bars + L::STAGES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (tc_smem(smem) & 1023u) {                               // the swizzled tiles need an aligned base
        if (threadIdx.x == 0) tc_fail(&g_attn_dec_f8_error, 9, ACORN_KERNEL_ATTN_DECODE_F8);
        return;
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < L::STAGES; ++s) { mbar_init(full0 + 8 * s, 33); mbar_init(empty0 + 8 * s, DF8_WARPS); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const bool cluster = !SHARES && dp.num_splits > 1;
    // every CTA of the cluster says that it runs; nobody writes into a peer's shared memory before all have
    if (cluster) cg::this_cluster().barrier_arrive();
    pdl_wait();
    pdl_trigger();

    F8Walk walk;
    const int split = SHARES ? 0 : blockIdx.y;
    if constexpr (SHARES) {
        int* before = reinterpret_cast<int*>(smem + L::RECV);
        int4* tiles = reinterpret_cast<int4*>(smem + L::RECV + (DF8_SHARE_TILES + 4) * 4);
        for (int k = threadIdx.x; k < dp.n_tiles; k += DF8_THREADS) {
            const F8Tile t(dp, k);
            before[k + 1] = t.n_chunks;
            tiles[k] = make_int4(t.r, t.tok0, t.n_q, t.pos0);
        }
        __syncthreads();
        if (warp == 0) {
            int sum = 0;
            for (int t0 = 0; t0 < dp.n_tiles; t0 += 32) {
                int v = t0 + lane < dp.n_tiles ? before[t0 + lane + 1] : 0;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const int w = __shfl_up_sync(0xffffffffu, v, o);
                    if (lane >= o) v += w;
                }
                if (t0 + lane < dp.n_tiles) before[t0 + lane + 1] = sum + v;
                sum += __shfl_sync(0xffffffffu, v, 31);
            }
            if (lane == 0) before[0] = 0;
        }
        __syncthreads();
        const int64_t total = (int64_t)before[dp.n_tiles] * p.nkv;
        const int64_t share = max((int64_t)DF8_SHARE_MIN, (total + gridDim.x - 1) / gridDim.x);
        walk.before = before;
        walk.tiles = tiles;
        walk.n_tiles = dp.n_tiles;
        walk.nkv = p.nkv;
        walk.at = min(total, blockIdx.x * share);
        walk.end = min(total, walk.at + share);
        if (blockIdx.x == 0) {
            for (int k = threadIdx.x; k < dp.n_tiles; k += DF8_THREADS)
                dp.plan[k] = make_int4(before[k], before[k + 1] - before[k], tiles[k].y, tiles[k].z);
            if (threadIdx.x == 0) dp.plan[dp.n_tiles] = make_int4((int)min(share, (int64_t)0x7fffffff), 0, 0, 0);
        }
    }
    const int rep = p.nq / p.nkv;
    const int g = lane >> 2, i = lane & 3;
    const int log_box = min(p.logP, 6);
    // the parts this CTA takes; fn(tile, kv head, first chunk, end, whether the share begins with it)
    auto parts = [&](auto fn) {
        if constexpr (SHARES) {
            for (bool first = true; walk.next(); first = false)
                if (!fn(F8Tile(p, walk.tiles[walk.ti]), walk.kvh, walk.c0, walk.c1, first)) break;
        } else {
            const F8Tile t(dp, blockIdx.z);
            const int per = (t.n_chunks + dp.num_splits - 1) / dp.num_splits;
            const int c0 = min(t.n_chunks, split * per);
            fn(t, (int)blockIdx.x, c0, min(t.n_chunks, c0 + per), true);
        }
    };

    if (warp == DF8_WARPS) {
        // ---------------------------------------------------------------- producer
        // The whole warp: lane l looks up the cache row of keys 2 l and 2 l + 1 of a chunk, a chunk ahead of the loads, and
        // copies their exponents; an elected lane issues the boxes (one page, or 64 keys of a larger one).
        const int box = 1 << log_box;
        int n = 0;                                                // chunks so far
        parts([&](const F8Tile& t, int kvh, int c0, int c1, bool) -> bool {
            const int* table = p.block_table + (int64_t)t.r * p.table_stride - p.page_base[t.r];
            const int first_key = p.page_base[t.r] << p.logP;
            auto row_at = [&](int c) -> int {
                const int key = t.key0(c) + 2 * lane;
                int b = key & ~(box - 1);
                if (b >= t.hi) b = (t.hi - 1) & ~(box - 1);       // masked later: any box that exists
                if (b < first_key) b = first_key;
                const int page = table[b >> p.logP];
                return ((page * p.nkv + kvh) << p.logP) + (b & ((1 << p.logP) - 1)) + (key & (box - 1));
            };
            int row_next = c0 < c1 ? row_at(c0) : 0;
            for (int c = c0; c < c1; ++c, ++n) {
                const int row = row_next, s = n % L::STAGES;
                if (c + 1 < c1) row_next = row_at(c + 1);
                const bool got = mbar_wait(empty0 + 8 * s, ((n / L::STAGES) & 1) ^ 1);
                if (!got && lane == 0) tc_fail(&g_attn_dec_f8_error, 1, ACORN_KERNEL_ATTN_DECODE_F8);
                if (!__all_sync(0xffffffffu, got)) return false;
                if (elect_one()) mbar_expect_tx(full0 + 8 * s, L::STAGE_BYTES);
                cp_async_bytes<4>(tc_smem(smem + L::SCALES + s * L::SCALE_BYTES) + 4 * lane, p.scales + 2 * (int64_t)row);
                cp_async_arrive(full0 + 8 * s);
                for (int k = 0; k < DF8_CHUNK; k += box) {
                    const int y = __shfl_sync(0xffffffffu, row, k >> 1);
                    if (elect_one()) {
                        const uint32_t dst = tc_smem(smem + s * L::STAGE_BYTES) + (uint32_t)(2 * k * D);
                        tma_load_3d(dst, &map_k, full0 + 8 * s, 0, y, 0);
                        if (!dp.joint) tma_load_3d(dst + box * D, &map_v, full0 + 8 * s, 0, y, 0);
                    }
                }
            }
            return true;
        });
        // the last stages' copies have landed before the CTA ends, also where the compute warps gave up
        for (int k = max(0, n - L::STAGES); k < n; ++k) mbar_wait(full0 + 8 * (k % L::STAGES), (k / L::STAGES) & 1);
        if (cluster) {
            cg::this_cluster().barrier_wait();
            cg::this_cluster().sync();
        }
        return;
    }

    // -------------------------------------------------------------------- compute warps
    // this lane's pieces of a stage: keys g and g + 8, values of keys 2 i, 2 i + 1, 8 + 2 i, 9 + 2 i of the warp's 16
    const int k_skip = dp.v_first ? 1 << log_box : 0, v_skip = (1 << log_box) - k_skip;
    uint32_t k_at[2], v_at[4];
#pragma unroll
    for (int k = 0; k < 2; ++k) k_at[k] = L::at(f8_stage_row(warp * 16 + 8 * k + g, log_box) + k_skip, (WORDS / 4) * i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int row = f8_stage_row(warp * 16 + 2 * i + (k & 1) + 8 * (k >> 1), log_box) + v_skip;
        v_at[k] = D == 128 ? L::at(row, g) : L::at(row, g >> 1) + 8 * (g & 1);
    }
    int n = 0;                                                    // chunks so far
    parts([&](const F8Tile& t, int kvh, int c0, int c1, bool first) -> bool {
        const int m_rows = t.n_q * rep, tok0 = t.tok0;
        float o[NH][WORDS][4];
        float m_ref[NH][2], t_ref[NH][2], l_run[NH][2];
        // queries: this lane holds row g (of each half), entries i * D / 4 .. + D / 4 - 1 of the head, as the B operand
        uint32_t qb[NH][WORDS][2];
        float factor[NH][2];                                      // of query rows 2 i and 2 i + 1: the softmax scale, and what undoes
                                                                  // the row's power of two
        int qpos[NH][2], first_seen[NH][2];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            const int m = 8 * h + g;
            const bool live = m < m_rows;
            const int j = live ? m / rep : 0;
            const uint4* src = reinterpret_cast<const uint4*>(p.q + (int64_t)(tok0 + j) * p.q_stride +
                                                              (int64_t)(kvh * rep + (live ? m - j * rep : 0)) * D + i * (D / 4));
            uint32_t w[2 * WORDS];
#pragma unroll
            for (int k = 0; k < WORDS / 2; ++k) {
                const uint4 v = live ? src[k] : make_uint4(0u, 0u, 0u, 0u);
                w[4 * k] = v.x; w[4 * k + 1] = v.y; w[4 * k + 2] = v.z; w[4 * k + 3] = v.w;
            }
            float most = 0.f;
#pragma unroll
            for (int k = 0; k < 2 * WORDS; ++k)
                most = fmaxf(most, fmaxf(fabsf(__uint_as_float(w[k] << 16)), fabsf(__uint_as_float(w[k] & 0xffff0000u))));
            most = quad_max(most);
            // 2^14 <= most * 2^up < 2^15; rows of zeros and of numbers that are none as they are
            const int ex = (int)(__float_as_uint(most) >> 23) - 127;
            const int up = most == 0.f || ex == 128 ? 0 : min(126, 14 - ex);
            const float f = f8_pow2(up), back = f8_pow2(-up);
#pragma unroll
            for (int k = 0; k < WORDS; ++k)
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    qb[h][k][b] = pack_f16(__uint_as_float(w[2 * k + b] << 16) * f, __uint_as_float(w[2 * k + b] & 0xffff0000u) * f);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                factor[h][b] = __shfl_sync(0xffffffffu, back, 4 * (2 * i + b)) * p.scale_log2;
                qpos[h][b] = t.pos0 + min((8 * h + 2 * i + b) / rep, max(t.n_q - 1, 0));
                first_seen[h][b] = mask_lo(p.mask, qpos[h][b]);
                m_ref[h][b] = t_ref[h][b] = DF8_NONE;
                l_run[h][b] = 0.f;
            }
#pragma unroll
            for (int n = 0; n < WORDS; ++n) { o[h][n][0] = o[h][n][1] = o[h][n][2] = o[h][n][3] = 0.f; }
        }
        const int last_lo = mask_lo(p.mask, t.hi - 1);              // the last query's rule starts last
        bool good = true;
        for (int c = c0; c < c1; ++c, ++n) {
            const int s = n % L::STAGES;
            if (!mbar_wait(full0 + 8 * s, (n / L::STAGES) & 1)) {
                tc_fail(&g_attn_dec_f8_error, 2, ACORN_KERNEL_ATTN_DECODE_F8);
                good = false;
            }
            good = __all_sync(0xffffffffu, good);
            if (!good) break;
            const int wkey0 = t.key0(c) + warp * 16;             // first key of this warp's 16
            if (wkey0 < t.hi && (wkey0 + 15 >= t.lo || wkey0 < p.mask.keep)) {
                const uint8_t* stage = smem + s * L::STAGE_BYTES;
                float sc[NH][4], sd[NH][4];                       // two chains of products
#pragma unroll
                for (int h = 0; h < NH; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[h][e] = sd[h][e] = 0.f;
                uint32_t kw[2][WORDS];                            // codes of keys g and g + 8
#pragma unroll
                for (int r2 = 0; r2 < 2; ++r2)
#pragma unroll
                    for (int q = 0; q < WORDS / 4; ++q) {
                        // pieces 2 i and 2 i + 1 differ in one bit, swizzled or not
                        const uint4 v = *reinterpret_cast<const uint4*>(stage + (k_at[r2] ^ (16 * q)));
                        kw[r2][4 * q] = v.x; kw[r2][4 * q + 1] = v.y; kw[r2][4 * q + 2] = v.z; kw[r2][4 * q + 3] = v.w;
                    }
                // exponents of keys g and g + 8: key byte, value byte
                const uint8_t* sp = smem + L::SCALES + s * L::SCALE_BYTES + 2 * (warp * 16 + g);
                const uint32_t sw[2] = {*reinterpret_cast<const uint16_t*>(sp), *reinterpret_cast<const uint16_t*>(sp + 16)};
#pragma unroll
                for (int k = 0; k < WORDS; ++k) {
                    const uint32_t a[4] = {f8_to_f16x2((uint16_t)kw[0][k]), f8_to_f16x2((uint16_t)kw[1][k]),
                                           f8_to_f16x2((uint16_t)(kw[0][k] >> 16)), f8_to_f16x2((uint16_t)(kw[1][k] >> 16))};
#pragma unroll
                    for (int h = 0; h < NH; ++h) mma_f16_16816(k & 1 ? sd[h] : sc[h], a, qb[h][k][0], qb[h][k][1]);
                }
                // all of the tile's queries see all 16 keys: no mask
                const bool whole = wkey0 + 15 <= t.pos0 && wkey0 >= last_lo;
                float ve[2], ks[2];
#pragma unroll
                for (int r2 = 0; r2 < 2; ++r2) {
                    const uint32_t kbyte = sw[r2] & 255u, vbyte = sw[r2] >> 8;
                    ks[r2] = vbyte == F8_NAN_BYTE ? f8_scale(vbyte) : f8_scale(kbyte);
                    ve[r2] = (float)((int)vbyte - 127);
                }
                bool grew = false;
                float mx[NH][2], tx[NH][2];
#pragma unroll
                for (int h = 0; h < NH; ++h)
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
#pragma unroll
                        for (int r2 = 0; r2 < 2; ++r2) {
                            float x = (sc[h][2 * r2 + b] + sd[h][2 * r2 + b]) * factor[h][b] * ks[r2];
                            if (!whole) {
                                const int key = wkey0 + 8 * r2 + g;
                                if (!(key <= qpos[h][b] && (key >= first_seen[h][b] || key < p.mask.keep))) x = -INFINITY;
                            }
                            sc[h][2 * r2 + b] = x;
                        }
                        mx[h][b] = fmaxf(sc[h][b] + ve[0], sc[h][2 + b] + ve[1]);
                        tx[h][b] = fmaxf(sc[h][b], sc[h][2 + b]);
                        grew = grew || mx[h][b] > m_ref[h][b] + DF8_GROW_LOG2 || tx[h][b] > t_ref[h][b] + DF8_SUM_LOG2;
                    }
                if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                    for (int h = 0; h < NH; ++h)
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const float top = column_max(mx[h][b]);
                            if (top > m_ref[h][b]) {
                                const float corr = fast_exp2(m_ref[h][b] - top);          // from DF8_NONE: 0
                                m_ref[h][b] = top;
#pragma unroll
                                for (int n2 = 0; n2 < WORDS; ++n2) { o[h][n2][b] *= corr; o[h][n2][2 + b] *= corr; }
                            }
                            const float most = column_max(tx[h][b]);
                            if (most > t_ref[h][b]) {
                                l_run[h][b] *= fast_exp2(t_ref[h][b] - most);
                                t_ref[h][b] = most;
                            }
                        }
                }
                uint32_t pb[NH][2];                               // P as the B operand: query row g, keys 2 i.. and 8 + 2 i..
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    float w[4];
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int r2 = 0; r2 < 2; ++r2) {
                            l_run[h][b] += fast_exp2(sc[h][2 * r2 + b] - t_ref[h][b]);
                            w[2 * r2 + b] = fast_exp2(sc[h][2 * r2 + b] - m_ref[h][b] + ve[r2]);
                        }
                    pb[h][0] = movmatrix_trans(pack_f16(w[0], w[1]));
                    pb[h][1] = movmatrix_trans(pack_f16(w[2], w[3]));
                }
                // value codes of keys 2 i, 2 i + 1, 8 + 2 i, 9 + 2 i: entries g * D / 8 .. + D / 8 - 1 of each
                uint32_t vw[4][WORDS / 2];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if constexpr (D == 128) {
                        const uint4 v = *reinterpret_cast<const uint4*>(stage + v_at[k]);
                        vw[k][0] = v.x; vw[k][1] = v.y; vw[k][2] = v.z; vw[k][3] = v.w;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2*>(stage + v_at[k]);
                        vw[k][0] = v.x; vw[k][1] = v.y;
                    }
                }
                if (!whole) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int key = wkey0 + 2 * i + (k & 1) + 8 * (k >> 1);
                        if (!(key < t.hi && (key >= t.lo || key < p.mask.keep))) {
#pragma unroll
                            for (int w = 0; w < WORDS / 2; ++w) vw[k][w] = 0u;
                        }
                    }
                }
                // row tile n: entries g * D / 8 + 2 n (rows g) and the one after it (rows g + 8)
#pragma unroll
                for (int w = 0; w < WORDS / 2; ++w)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t x = __byte_perm(vw[0][w], vw[1][w], half ? 0x7362 : 0x5140);
                        const uint32_t y = __byte_perm(vw[2][w], vw[3][w], half ? 0x7362 : 0x5140);
                        const uint32_t a[4] = {f8_to_f16x2((uint16_t)x), f8_to_f16x2((uint16_t)(x >> 16)), f8_to_f16x2((uint16_t)y),
                                               f8_to_f16x2((uint16_t)(y >> 16))};
#pragma unroll
                        for (int h = 0; h < NH; ++h) mma_f16_16816(o[h][2 * w + half], a, pb[h][0], pb[h][1]);
                    }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty0 + 8 * s);
        }
#pragma unroll
        for (int h = 0; h < NH; ++h) { l_run[h][0] = column_sum(l_run[h][0]); l_run[h][1] = column_sum(l_run[h][1]); }
        // ---- the warps joined
        float* sm_m = reinterpret_cast<float*>(smem + L::MERGE);  // [WARPS][ROWS]
        float* sm_t = sm_m + ROWS * DF8_WARPS;
        float* sm_l = sm_t + ROWS * DF8_WARPS;
        float* sm_o = sm_l + ROWS * DF8_WARPS;                    // [WARPS][ROWS][D]
        good = compute_all(good);                                 // the part before has been read; a wait that gave up ends the walk of all
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int m = warp * ROWS + 8 * h + 2 * i + b;
                if (g == 0) {
                    sm_m[m] = m_ref[h][b];
                    sm_t[m] = t_ref[h][b];
                    sm_l[m] = l_run[h][b];
                }
#pragma unroll
                for (int n2 = 0; n2 < WORDS; n2 += 2)
                    *reinterpret_cast<float4*>(sm_o + m * D + g * (D / 8) + 2 * n2) =
                        make_float4(o[h][n2][b], o[h][n2][2 + b], o[h][n2 + 1][b], o[h][n2 + 1][2 + b]);
            }
        compute_all(true);
        // received partial rows: recv[rank of the sender][slot][RECV_ROW]
        float* recv = reinterpret_cast<float*>(smem + L::RECV);
        const int csize = cluster ? dp.num_splits : 1;
        const int slots = (dp.tile_tokens * rep + csize - 1) / csize;
        const bool whole_pair = SHARES ? c0 == 0 && c1 == t.n_chunks : !cluster;
        if (cluster) cg::this_cluster().barrier_wait();
        for (int m = warp; m < m_rows; m += DF8_WARPS) {          // a warp a row, D / 32 neighbouring entries a lane
            constexpr int E = D / 32;
            const int head = kvh * rep + m % rep;
            const float sink = p.sink && c0 == 0 && split == 0 ? p.sink[head] * 1.4426950408889634f : -INFINITY;
            float mstar = DF8_NONE, tstar = fmaxf(DF8_NONE, sink);
#pragma unroll
            for (int w = 0; w < DF8_WARPS; ++w) {
                mstar = fmaxf(mstar, sm_m[w * ROWS + m]);
                tstar = fmaxf(tstar, sm_t[w * ROWS + m]);
            }
            float sum = sink == -INFINITY ? 0.f : exp2f(sink - tstar);
            F8Floats<E> mean = {};
#pragma unroll
            for (int w = 0; w < DF8_WARPS; ++w) {                 // a warp without keys has a sum and an output of 0
                sum += exp2f(sm_t[w * ROWS + m] - tstar) * sm_l[w * ROWS + m];
                const float f = exp2f(sm_m[w * ROWS + m] - mstar);
                const F8Floats<E> part = reinterpret_cast<const F8Floats<E>*>(sm_o + (w * ROWS + m) * D)[lane];
#pragma unroll
                for (int e = 0; e < E; ++e) mean.v[e] += f * part.v[e];
            }
            const bool empty = sum == 0.f;                        // no key of this part is seen by the query
            const float back = exp2f(0.5f * (mstar - tstar));     // in two steps: 2^(m - r) alone may not be a float
#pragma unroll
            for (int e = 0; e < E; ++e) mean.v[e] = empty && !whole_pair ? 0.f : mean.v[e] / sum * back * back;
            if (whole_pair) {
                __nv_bfloat162* dst = reinterpret_cast<__nv_bfloat162*>(p.out + ((int64_t)(tok0 + m / rep) * p.nq + head) * D + E * lane);
#pragma unroll
                for (int e = 0; e < E; e += 2) dst[e / 2] = __floats2bfloat162_rn(mean.v[e], mean.v[e + 1]);
            } else if (cluster) {
                // to the CTA that finishes this row; a split without keys sends a log-sum of -inf
                const uint32_t dst = cluster_map(tc_smem(recv + (split * slots + m / csize) * L::RECV_ROW), m % csize);
                st_cluster(dst + 4 * E * lane, mean);
                if (lane == 0) st_cluster_f32(dst + 4 * D, empty ? -INFINITY : tstar + log2f(sum));
            } else {
                const int64_t at = ((int64_t)blockIdx.x * 2 + (first ? 0 : 1)) * ROWS + m;
                reinterpret_cast<F8Floats<E>*>(dp.part_o + at * D)[lane] = mean;
                if (lane == 0) dp.part_lse[at] = empty ? -INFINITY : tstar + log2f(sum);
            }
        }
        if (cluster) {
            cg::this_cluster().sync();                            // all partial rows have arrived
            for (int idx = threadIdx.x; idx < slots * D; idx += 32 * DF8_WARPS) {
                const int slot = idx / D, e = idx - slot * D;
                const int m = split + slot * csize;               // the rows this CTA finishes: rank, rank + csize, ...
                if (m >= m_rows) break;
                float mstar = -INFINITY;
                for (int s = 0; s < csize; ++s) mstar = fmaxf(mstar, recv[(s * slots + slot) * L::RECV_ROW + D]);
                float sum = 0.f, acc = 0.f;
                for (int s = 0; s < csize; ++s) {
                    const float lse = recv[(s * slots + slot) * L::RECV_ROW + D];
                    const float f = lse == -INFINITY ? 0.f : exp2f(lse - mstar);
                    sum += f;
                    acc += f * recv[(s * slots + slot) * L::RECV_ROW + e];
                }
                p.out[((int64_t)(tok0 + m / rep) * p.nq + kvh * rep + m % rep) * D + e] = __float2bfloat16_rn(acc / sum);
            }
        }
        return good;
    });
}

// Even shares: the pairs that several CTAs had parts of.  One CTA per (tile, kv head, query row); its four warps take every
// fourth part, D / 32 entries a lane.
template <int D, int NH>
__global__ void __launch_bounds__(128) attention_decode_f8_join_kernel(const DecodeF8Params dp) {
    constexpr int ROWS = 8 * NH, E = D / 32;
    __shared__ float so[4][D], sl[4], sm[4];
    pdl_wait();
    pdl_trigger();
    const F8AttnParams& p = dp.a;
    const int kvh = blockIdx.x, m = blockIdx.y, rep = p.nq / p.nkv;
    const int4 t = dp.plan[blockIdx.z];                            // chunks before, chunks, first token, tokens
    const int share = dp.plan[dp.n_tiles].x;
    const int64_t u0 = (int64_t)t.x * p.nkv + (int64_t)kvh * t.y;
    if (t.y == 0 || m >= t.w * rep) return;
    // (64-bit quotients take a hundred instructions, and nearly every call's chunks fit 32 bits)
    const bool narrow = u0 + t.y < 0x7fffffff;
    const int b0 = narrow ? (int)u0 / share : (int)(u0 / share);
    const int b1 = narrow ? ((int)u0 + t.y - 1) / share : (int)((u0 + t.y - 1) / share);
    if (b0 == b1) return;                                         // one CTA had it all
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // the first CTA's part is the last of its share, unless its share begins with the pair; the others begin theirs with it
    const int begun = (int64_t)b0 * share < u0 ? 1 : 0;
    auto at = [&](int b) { return (b * 2 + (b == b0 ? begun : 0)) * ROWS + m; };
    float top = -INFINITY, sum = 0.f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int c = b0 + warp; c <= b1; c += 4 * 4) {                // four parts at a time, all on their way together
        float lse[4], v[4][E];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool live = c + 4 * k <= b1;
            lse[k] = live ? dp.part_lse[at(c + 4 * k)] : -INFINITY;
#pragma unroll
            for (int e = 0; e < E; ++e) v[k][e] = live ? dp.part_o[at(c + 4 * k) * D + lane * E + e] : 0.f;
        }
        float mx = top;
#pragma unroll
        for (int k = 0; k < 4; ++k) mx = fmaxf(mx, lse[k]);
        const float corr = top == -INFINITY ? 0.f : exp2f(top - mx);
        top = mx;
        sum *= corr;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= corr;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float f = lse[k] == -INFINITY ? 0.f : exp2f(lse[k] - top);
            sum += f;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = fmaf(f, v[k][e], acc[e]);
        }
    }
    if (lane == 0) { sm[warp] = top; sl[warp] = sum; }
#pragma unroll
    for (int e = 0; e < E; ++e) so[warp][lane * E + e] = acc[e];
    __syncthreads();
    const float all = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float f[4], total = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = sm[w] == -INFINITY ? 0.f : exp2f(sm[w] - all);
        total += f[w] * sl[w];                                    // (a part whose logarithm is NaN left a sum that is NaN)
    }
    for (int e = threadIdx.x; e < D; e += 128)
        p.out[((int64_t)(t.z + m / rep) * p.nq + kvh * rep + m % rep) * D + e] =
            __float2bfloat16_rn((f[0] * so[0][e] + f[1] * so[1][e] + f[2] * so[2][e] + f[3] * so[3][e]) / total);
}

// What this kernel takes.
extern "C" int acorn_attention_decode_f8_supported(int nq, int nkv, int d, int P) {
    return nkv > 0 && nq % nkv == 0 && nq / nkv <= 16 && (d == 64 || d == 128) && P >= 8 && P <= 4096 && (P & (P - 1)) == 0;
}

template <int D, int NH, bool SHARES>
static cudaError_t configure_decode_f8(size_t smem) {
    static AcornPerDevice configured;
    if (configured.seen()) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(attention_decode_f8_kernel<D, NH, SHARES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess && !SHARES)
        e = cudaFuncSetAttribute(attention_decode_f8_kernel<D, NH, SHARES>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) configured.mark();
    return e;
}

// CTAs of the even shares: as many as the device holds at once.
template <int D, int NH> static int share_ctas() {
    static int ctas[64] = {};
    const int dev = AcornPerDevice::current();
    if (dev < 0) return 0;
    if (ctas[dev] == 0) {
        int per_sm = 0;
        const size_t smem = DecodeF8<D, NH>::RECV + DecodeF8<D, NH>::SHARES;
        if (configure_decode_f8<D, NH, true>(smem) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, attention_decode_f8_kernel<D, NH, true>, DF8_THREADS, smem) != cudaSuccess)
            return 0;
        ctas[dev] = per_sm * acorn_sms();
    }
    return ctas[dev];
}

// CTAs that share the work of a call with num_splits 0 (its scratch: part_o [CTAs, 2, rows, d], part_lse [CTAs, 2, rows] float32,
// plan [n_tiles + 1, 4] int32, with rows = 8 up to 8 query rows a tile, else 16); 0 where there are too many tiles for that.
extern "C" int acorn_attention_decode_f8_shares(int nq, int nkv, int d, int tile_tokens, int n_tiles) {
    if (n_tiles > DF8_SHARE_TILES || nkv < 1 || nq % nkv) return 0;
    const bool one = tile_tokens * (nq / nkv) <= 8;
    if (d == 128) return one ? share_ctas<128, 1>() : share_ctas<128, 2>();
    return one ? share_ctas<64, 1>() : share_ctas<64, 2>();
}

template <int D, int NH>
static int launch_decode_f8(DecodeF8Params dp, int64_t num_pages, cudaStream_t stream) {
    using L = DecodeF8<D, NH>;
    const F8AttnParams& p = dp.a;
    CUtensorMap mk, mv;
    const int P = 1 << p.logP, box_rows = P < DF8_CHUNK ? P : DF8_CHUNK;
    const int rc = make_code_maps(&mk, &mv, p, num_pages, D, box_rows,
                                  D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, &dp.joint, &dp.v_first);
    if (rc) return rc;
    if (dp.num_splits == 0) {
        const int ctas = share_ctas<D, NH>();
        if (ctas < 1) return ACORN_ERR_UNSUPPORTED;
        const int e = acorn_launch(attention_decode_f8_kernel<D, NH, true>, dim3(ctas), dim3(DF8_THREADS), (size_t)(L::RECV + L::SHARES), stream,
                                   mk, mv, dp);
        return e ? e : acorn_launch(attention_decode_f8_join_kernel<D, NH>, dim3(p.nkv, dp.tile_tokens * (p.nq / p.nkv), dp.n_tiles),
                                    dim3(128), 0, stream, dp);
    }
    const int rows = dp.tile_tokens * (p.nq / p.nkv), splits = dp.num_splits;
    const size_t recv = splits > 1 ? (size_t)splits * ((rows + splits - 1) / splits) * L::RECV_ROW * 4 : 0;
    cudaError_t e = configure_decode_f8<D, NH, false>(L::RECV + (size_t)32 * L::RECV_ROW * 4);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.nkv, splits, dp.n_tiles);
    cfg.blockDim = dim3(DF8_THREADS);
    cfg.dynamicSmemBytes = L::RECV + recv;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = splits;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = acorn_pdl_enabled() ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, attention_decode_f8_kernel<D, NH, false>, mk, mv, dp);
    return e != cudaSuccess ? (int)e : acorn_launch_status();
}

// num_splits: 1 to 8 or 16 (a cluster joins them), or 0: even shares, which need the scratch of acorn_attention_decode_f8_shares.
extern "C" int acorn_attention_decode_f8(const void* q, int64_t q_stride, void* out, const void* k_pages, const void* v_pages,
                                         const void* scales, int64_t num_pages, const int* block_table, const int* page_base,
                                         int table_stride, const int* row_start, const int* row_pos, const int* tiles, int n_tiles,
                                         int nq, int nkv, int d, int P, float scale, int window, int chunk, int keep,
                                         const float* sink, int tile_tokens, int num_splits, float* part_o, float* part_lse, void* plan,
                                         cudaStream_t stream) {
    if (n_tiles <= 0) return 0;
    if (!acorn_attention_decode_f8_supported(nq, nkv, d, P) || n_tiles > 65535 || q_stride % 8 || num_splits < 0 ||
        (num_splits > 8 && num_splits != DF8_CLUSTER_MAX) || tile_tokens < 1 || tile_tokens > 16 / (nq / nkv) || nkv > 65535)
        return ACORN_ERR_UNSUPPORTED;
    if (num_splits == 0 && (n_tiles > DF8_SHARE_TILES || part_o == nullptr || part_lse == nullptr || plan == nullptr))
        return ACORN_ERR_UNSUPPORTED;
    DecodeF8Params dp;
    F8AttnParams& p = dp.a;
    p.q = (const bf16*)q; p.q_stride = q_stride; p.out = (bf16*)out; p.k_pages = (const uint8_t*)k_pages;
    p.v_pages = (const uint8_t*)v_pages; p.scales = (const uint8_t*)scales; p.block_table = block_table; p.page_base = page_base;
    p.row_start = row_start; p.row_pos = row_pos; p.tiles = tiles; p.sink = sink; p.table_stride = table_stride;
    p.nq = nq; p.nkv = nkv; p.mask = {window, chunk, keep}; p.scale_log2 = scale * 1.4426950408889634f;
    p.logP = acorn_log2_exact_tc(P);
    dp.n_tiles = n_tiles; dp.tile_tokens = tile_tokens; dp.num_splits = num_splits;
    dp.part_o = part_o; dp.part_lse = part_lse; dp.plan = (int4*)plan;
    const bool one = tile_tokens * (nq / nkv) <= 8;
    if (d == 128) return one ? launch_decode_f8<128, 1>(dp, num_pages, stream) : launch_decode_f8<128, 2>(dp, num_pages, stream);
    return one ? launch_decode_f8<64, 1>(dp, num_pages, stream) : launch_decode_f8<64, 2>(dp, num_pages, stream);
}

extern "C" int acorn_attention_decode_f8_error() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_attn_dec_f8_error, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_attn_dec_f8_error, &zero, sizeof(int));
    return v;
}

ACORN_ERROR_WORD_SETTER(acorn_attention_decode_f8_set_error_word)
