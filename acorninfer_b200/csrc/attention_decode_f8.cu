// Attention of few tokens a row over the pages of the 8-bit cache (f8_cache.cuh), head sizes 64 and 128: split-K flash decoding.
//
// One CTA per (tile, kv head, split).  A tile is up to 16 / rep tokens of one row (rep = nq / nkv query heads share a kv head);
// its (token, head) pairs are the 16 rows of an m16n8k16 tile, so the tokens of a tile read their row's pages together.
// A producer warp brings K and V codes by TMA (one box a page and head, swizzled) and their exponents by bulk copies into a ring of
// stages of 64 keys; each of the four other warps takes 16 keys of a stage:
//   S = Q K^T   codes become half-precision numbers by one conversion a pair (e4m3 is exact in it); the queries are
//               brought to half precision by a power of two per row (their largest entry to 2^14 .. 2^15, so that a bfloat16
//               entry is exact unless it is 2^-28 of the largest), and both powers of two meet the score in float32.
//   P = 2^(t + e_v - m)   t the score in units of log2, e_v the exponent of the key's value row, m the running maximum of t + e_v:
//               the value's power of two rides in the exponent, so that a weight is at most 1 (2^8 before the reference moves) in
//               half precision, with 11 bits where bfloat16 would keep 8, whatever the sizes of the value rows.
//   O += P V    on value codes as half-precision numbers; the denominator sums 2^(t - m) in float32.
// The layouts of the fragments are chosen so that a lane's codes are whole 16-byte pieces of rows: the order of the head's
// entries in a product of K is free (Q is laid out the same way), and so is the order of the output's columns.
// Codes of keys that no query of the tile reads are replaced by zeros (a slot that was never written may hold anything).
//
// The warps are merged through shared memory, the splits of a (tile, kv head) by a thread-block cluster through
// distributed shared memory (2 to 8, or 16 of them), more by a second kernel through scratch.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "f8_cache.cuh"
#include "mma_helpers.cuh"
#include "tcgen05_helpers.cuh"

namespace cg = cooperative_groups;

#define DF8_WARPS 4                         // compute warps; one more brings the codes
#define DF8_THREADS (32 * DF8_WARPS + 32)
#define DF8_CHUNK (16 * DF8_WARPS)
#define DF8_CLUSTER_MAX 16
#define DF8_GROW_LOG2 8.f                   // the reference maximum moves when a row's maximum outgrew it by more than this

__device__ int g_attn_dec_f8_error = 0;

struct DecodeF8Params {
    F8AttnParams a;
    int tile_tokens, num_splits, cluster_merge;
    float* part_o;            // [n_tiles, nkv, splits, 16, D]  (more splits than a cluster merges)
    float* part_lse;          // [n_tiles, nkv, splits, 16]
};

template <int D> struct DecodeF8 {
    static constexpr int STAGES = D == 128 ? 4 : 8;
    static constexpr int ROWS_BYTES = DF8_CHUNK * D;                  // the codes of a stage's keys (or values)
    static constexpr int STAGE_BYTES = 2 * ROWS_BYTES;
    static constexpr int SCALE_BYTES = 2 * DF8_CHUNK;
    static constexpr int RECV_ROW = D + 4;                            // floats a received partial row takes: the output, then its log-sum
    static constexpr int RING = STAGES * STAGE_BYTES;
    static constexpr int MERGE = (2 * DF8_WARPS * 16 + DF8_WARPS * 16 * D) * 4;
    static constexpr int BARS = RING > MERGE ? RING : MERGE;          // offsets in shared memory
    static constexpr int SCALES = BARS + 2 * STAGES * 8;
    static constexpr int RECV = SCALES + STAGES * SCALE_BYTES;
    // byte offset of the 16-byte piece `seg` of row `key` in a stage's region, as the TMA's swizzle places it
    static __device__ __forceinline__ uint32_t at(int key, int seg) {
        return D == 128 ? (uint32_t)(key * 128 + ((seg ^ (key & 7)) << 4)) : (uint32_t)(key * 64 + ((seg ^ ((key >> 1) & 3)) << 4));
    }
};

__device__ __forceinline__ void mma_f16_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}

// Untiled bulk copy global -> shared (16-byte aligned, a multiple of 16 bytes).
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

template <int D>
__global__ void __launch_bounds__(DF8_THREADS) attention_decode_f8_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                         const __grid_constant__ CUtensorMap map_v,
                                                                         const DecodeF8Params dp) {
    using L = DecodeF8<D>;
    constexpr int WORDS = D / 16;                              // 32-bit words of codes a lane holds of a key row; k-steps of a product
    constexpr int NT = D / 8;                                  // column tiles of the output
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
        for (int s = 0; s < L::STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, DF8_WARPS); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // every CTA of the cluster says that it runs; nobody writes into a peer's shared memory before all have
    if (dp.cluster_merge) cg::this_cluster().barrier_arrive();
    pdl_wait();
    pdl_trigger();

    const int kvh = blockIdx.x, split = blockIdx.y, ti = blockIdx.z;
    const int r = p.tiles[2 * ti], q0 = p.tiles[2 * ti + 1];
    const int rep = p.nq / p.nkv;
    const int tok0 = p.row_start[r] + q0;
    const int n_q = max(0, min(dp.tile_tokens, p.row_start[r + 1] - tok0));
    const int m_rows = n_q * rep;
    const int pos0 = p.row_pos[r] + q0;
    const int hi = pos0 + n_q;                                  // keys < hi are read by the tile
    const int lo = mask_lo(p.mask, pos0);                       // the first query's rule starts first
    const int base_key = lo & ~(DF8_CHUNK - 1);                 // chunks start at multiples of 64 keys
    // the kept first keys, where the rule's range starts beyond them, are chunks of their own in front
    const int nkb = (p.mask.keep > 0 && base_key > 0) ? min((p.mask.keep + DF8_CHUNK - 1) / DF8_CHUNK, base_key / DF8_CHUNK) : 0;
    const int n_chunks = n_q > 0 ? nkb + (hi - base_key + DF8_CHUNK - 1) / DF8_CHUNK : 0;
    const int per = (n_chunks + dp.num_splits - 1) / dp.num_splits;
    const int c0 = min(n_chunks, split * per), c1 = min(n_chunks, c0 + per);
    auto key0_of = [&](int c) { return c < nkb ? c * DF8_CHUNK : base_key + (c - nkb) * DF8_CHUNK; };

    float o[NT][4];
    float m_ref[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
    const int g = lane >> 2, i = lane & 3;

    if (warp == DF8_WARPS) {
        // ---------------------------------------------------------------- producer
        // The whole warp: lane l looks up the cache rows of the l-th box (one page, or 64 keys of a larger one) of a batch of
        // 32, a batch ahead of the loads; an elected lane issues the loads.
        const int* table = p.block_table + (int64_t)r * p.table_stride - p.page_base[r];
        const int P = 1 << p.logP;
        const int rows_per_op = P < DF8_CHUNK ? P : DF8_CHUNK;
        const int log_ops = 6 - (p.logP < 6 ? p.logP : 6);       // boxes a chunk: 64 / rows_per_op
        const int n_ops = (c1 - c0) << log_ops;
        const int first_key = p.page_base[r] << p.logP;
        auto row_of = [&](int idx) -> int {
            const int b = idx < n_ops ? idx : 0;
            int key = key0_of(c0 + (b >> log_ops)) + (b & ((1 << log_ops) - 1)) * rows_per_op;
            if (key >= hi) key = hi - 1 - ((hi - 1) & (rows_per_op - 1));        // masked later: any rows that exist
            if (key < first_key) key = first_key;
            const int page = table[key >> p.logP];
            return ((page * p.nkv + kvh) << p.logP) + (key & (P - 1));
        };
        int rows_next = n_ops > 0 ? row_of(lane) : 0;
        bool good = true;
        for (int b0 = 0; b0 < n_ops && good; b0 += 32) {
            const int rows_cur = rows_next;
            if (b0 + 32 < n_ops) rows_next = row_of(b0 + 32 + lane);
            const int n_here = min(32, n_ops - b0);
            for (int l = 0; l < n_here; ++l) {
                const int idx = b0 + l, n = idx >> log_ops, k = idx & ((1 << log_ops) - 1), s = n % L::STAGES;
                if (k == 0) {                                     // first box of a chunk: its stage must be free
                    const bool got = mbar_wait(empty0 + 8 * s, ((n / L::STAGES) & 1) ^ 1);
                    if (!got && lane == 0) tc_fail(&g_attn_dec_f8_error, 1, ACORN_KERNEL_ATTN_DECODE_F8);
                    good = __all_sync(0xffffffffu, got);
                    if (!good) break;
                    if (elect_one()) mbar_expect_tx(full0 + 8 * s, L::STAGE_BYTES + L::SCALE_BYTES);
                }
                const int row = __shfl_sync(0xffffffffu, rows_cur, l);
                if (elect_one()) {
                    const uint32_t dst = tc_smem(smem + s * L::STAGE_BYTES) + (uint32_t)(k * rows_per_op) * D;
                    tma_load_2d(dst, &map_k, full0 + 8 * s, 0, row);
                    tma_load_2d(dst + L::ROWS_BYTES, &map_v, full0 + 8 * s, 0, row);
                    bulk_load(tc_smem(smem + L::SCALES + s * L::SCALE_BYTES) + 2 * k * rows_per_op, p.scales + 2 * (int64_t)row,
                              2 * rows_per_op, full0 + 8 * s);
                }
            }
        }
    } else {
        // ---------------------------------------------------------------- compute warps
        // this lane's query entries: rows g and g + 8, entries i * D / 4 .. + D / 4 - 1 of the head
        uint32_t qa[WORDS][4];
        float back[2];                                            // what undoes the rows' powers of two
        int qpos[2], first_seen[2];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            const int m = g + 8 * hh;
            const bool live = m < m_rows;
            const int j = live ? m / rep : 0;
            qpos[hh] = pos0 + j;
            first_seen[hh] = mask_lo(p.mask, qpos[hh]);
            const uint4* src = reinterpret_cast<const uint4*>(p.q + (int64_t)(tok0 + j) * p.q_stride +
                                                              (int64_t)(kvh * rep + (m - j * rep)) * D + i * (D / 4));
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
            const float f = f8_pow2(up);
            back[hh] = f8_pow2(-up);
#pragma unroll
            for (int k = 0; k < WORDS; ++k)
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    qa[k][hh + 2 * b] = pack_f16(__uint_as_float(w[2 * k + b] << 16) * f, __uint_as_float(w[2 * k + b] & 0xffff0000u) * f);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) { o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f; }
        bool good = true;
        for (int c = c0; c < c1; ++c) {
            const int n = c - c0, s = n % L::STAGES;
            if (good && !mbar_wait(full0 + 8 * s, (n / L::STAGES) & 1)) {
                tc_fail(&g_attn_dec_f8_error, 2, ACORN_KERNEL_ATTN_DECODE_F8);
                good = false;
            }
            good = __all_sync(0xffffffffu, good);
            if (!good) break;
            const int wkey0 = key0_of(c) + warp * 16;             // first key of this warp's 16
            const int wlast = wkey0 + 15;
            const bool any = wkey0 < hi && (wlast >= lo || wkey0 < p.mask.keep);
            if (any) {
                const uint32_t kb = tc_smem(smem + s * L::STAGE_BYTES), vb = kb + L::ROWS_BYTES;
                float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
                uint32_t kw[2][WORDS];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int q = 0; q < WORDS / 4; ++q) {
                        const uint4 v = lds128(kb + L::at(warp * 16 + 8 * h + g, (WORDS / 4) * i + q));
                        kw[h][4 * q] = v.x; kw[h][4 * q + 1] = v.y; kw[h][4 * q + 2] = v.z; kw[h][4 * q + 3] = v.w;
                    }
#pragma unroll
                for (int k = 0; k < WORDS; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        mma_f16_16816(sc[h], qa[k], f8_to_f16x2((uint16_t)kw[h][k]), f8_to_f16x2((uint16_t)(kw[h][k] >> 16)));
                // exponents of this lane's keys (8 h + 2 i and the one after it): key byte, value byte, twice
                uint32_t sw[2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    sw[h] = *reinterpret_cast<const uint32_t*>(smem + L::SCALES + s * L::SCALE_BYTES + 2 * (warp * 16 + 8 * h + 2 * i));
                // all of the tile's queries see all 16 keys: no mask (the last query's rule starts last)
                const bool whole = wlast <= pos0 && wkey0 >= mask_lo(p.mask, pos0 + n_q - 1);
                float ve[2][2], mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const uint32_t kbyte = (sw[h] >> (16 * b)) & 255u, vbyte = (sw[h] >> (16 * b + 8)) & 255u;
                        const float ks = p.scale_log2 * f8_scale(vbyte == F8_NAN_BYTE ? vbyte : kbyte);
                        ve[h][b] = (float)((int)vbyte - 127);
#pragma unroll
                        for (int hh = 0; hh < 2; ++hh) {
                            float t = sc[h][2 * hh + b] * back[hh] * ks;
                            if (!whole) {
                                const int key = wkey0 + 8 * h + 2 * i + b;
                                if (!(key <= qpos[hh] && (key >= first_seen[hh] || key < p.mask.keep))) t = -INFINITY;
                            }
                            sc[h][2 * hh + b] = t;
                            mx[hh] = fmaxf(mx[hh], t + ve[h][b]);
                        }
                    }
                bool grew = false;
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    mx[hh] = quad_max(mx[hh]);
                    grew = grew || mx[hh] > m_ref[hh] + DF8_GROW_LOG2;
                }
                if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh) {
                        if (mx[hh] > m_ref[hh] + DF8_GROW_LOG2) {
                            const float corr = fast_exp2(m_ref[hh] - mx[hh]);          // from -inf: 0
                            m_ref[hh] = mx[hh];
                            l_run[hh] *= corr;
#pragma unroll
                            for (int n2 = 0; n2 < NT; ++n2) { o[n2][2 * hh] *= corr; o[n2][2 * hh + 1] *= corr; }
                        }
                    }
                }
                float neg[2];
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) neg[hh] = m_ref[hh] == -INFINITY ? 0.f : -m_ref[hh];
                uint32_t pa[4];                                   // P as the A operand: rows g, g + 8, keys 2 i.. and 8 + 2 i..
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh) {
                        const float a = sc[h][2 * hh] + neg[hh], b = sc[h][2 * hh + 1] + neg[hh];
                        l_run[hh] += fast_exp2(a) + fast_exp2(b);
                        pa[2 * h + hh] = pack_f16(fast_exp2(a + ve[h][0]), fast_exp2(b + ve[h][1]));
                    }
                // value codes of keys 2 i, 2 i + 1, 8 + 2 i, 9 + 2 i: entries g * D / 8 .. of each
                uint32_t vw[4][NT / 4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int row = warp * 16 + 2 * i + (k & 1) + 8 * (k >> 1);
                    if constexpr (D == 128) {
                        const uint4 v = lds128(vb + L::at(row, g));
                        vw[k][0] = v.x; vw[k][1] = v.y; vw[k][2] = v.z; vw[k][3] = v.w;
                    } else {
                        const uint2 v = lds64(vb + L::at(row, g >> 1) + 8 * (g & 1));
                        vw[k][0] = v.x; vw[k][1] = v.y;
                    }
                }
                if (!whole) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int key = wkey0 + 2 * i + (k & 1) + 8 * (k >> 1);
                        if (!(key < hi && (key >= lo || key < p.mask.keep))) {
#pragma unroll
                            for (int w = 0; w < NT / 4; ++w) vw[k][w] = 0u;
                        }
                    }
                }
#pragma unroll
                for (int w = 0; w < NT / 4; ++w) {
                    const uint32_t a0 = __byte_perm(vw[0][w], vw[1][w], 0x5140), a1 = __byte_perm(vw[0][w], vw[1][w], 0x7362);
                    const uint32_t b0 = __byte_perm(vw[2][w], vw[3][w], 0x5140), b1 = __byte_perm(vw[2][w], vw[3][w], 0x7362);
                    mma_f16_16816(o[4 * w], pa, f8_to_f16x2((uint16_t)a0), f8_to_f16x2((uint16_t)b0));
                    mma_f16_16816(o[4 * w + 1], pa, f8_to_f16x2((uint16_t)(a0 >> 16)), f8_to_f16x2((uint16_t)(b0 >> 16)));
                    mma_f16_16816(o[4 * w + 2], pa, f8_to_f16x2((uint16_t)a1), f8_to_f16x2((uint16_t)b1));
                    mma_f16_16816(o[4 * w + 3], pa, f8_to_f16x2((uint16_t)(a1 >> 16)), f8_to_f16x2((uint16_t)(b1 >> 16)));
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty0 + 8 * s);
        }
        l_run[0] = quad_sum(l_run[0]);
        l_run[1] = quad_sum(l_run[1]);
    }
    // every stage has been consumed (the compute warps waited for each); the ring is free for the merge
    __syncthreads();
    float* sm_m = reinterpret_cast<float*>(smem);                 // [WARPS][16]
    float* sm_l = sm_m + 16 * DF8_WARPS;
    float* sm_o = sm_l + 16 * DF8_WARPS;                          // [WARPS][16][D]
    if (warp < DF8_WARPS) {
        if (i == 0) {
            sm_m[warp * 16 + g] = m_ref[0];
            sm_m[warp * 16 + g + 8] = m_ref[1];
            sm_l[warp * 16 + g] = l_run[0];
            sm_l[warp * 16 + g + 8] = l_run[1];
        }
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int n = 0; n < NT; n += 4)
                    *reinterpret_cast<float4*>(sm_o + (warp * 16 + g + 8 * hh) * D + (2 * i + b) * NT + n) =
                        make_float4(o[n][2 * hh + b], o[n + 1][2 * hh + b], o[n + 2][2 * hh + b], o[n + 3][2 * hh + b]);
    }
    __syncthreads();
    // received partial rows: recv[rank of the sender][slot][RECV_ROW]
    float* recv = reinterpret_cast<float*>(smem + L::RECV);
    const int csize = dp.cluster_merge ? dp.num_splits : 1;
    const int slots = (dp.tile_tokens * rep + csize - 1) / csize;
    if (dp.cluster_merge) cg::this_cluster().barrier_wait();
    for (int idx = threadIdx.x; idx < m_rows * D; idx += DF8_THREADS) {
        const int m = idx / D, e = idx - m * D;
        const int head = kvh * rep + m % rep;
        const float sink = p.sink && split == 0 ? p.sink[head] * 1.4426950408889634f : -INFINITY;
        float mstar = sink;
#pragma unroll
        for (int w = 0; w < DF8_WARPS; ++w) mstar = fmaxf(mstar, sm_m[w * 16 + m]);
        float sum = sink == -INFINITY ? 0.f : exp2f(sink - mstar), acc = 0.f;
#pragma unroll
        for (int w = 0; w < DF8_WARPS; ++w) {
            // a warp without keys has maximum -inf and sum 0; one whose keys are all NaN a sum that is NaN
            const float mw = sm_m[w * 16 + m], lw = sm_l[w * 16 + m];
            const float f = mw == -INFINITY ? 0.f : exp2f(mw - mstar);
            sum += f * lw;
            acc += f * sm_o[(w * 16 + m) * D + e];
        }
        const bool empty = mstar == -INFINITY && sum == 0.f;      // no key of this split is seen by the query
        if (dp.num_splits == 1) {
            p.out[((int64_t)(tok0 + m / rep) * p.nq + head) * D + e] = __float2bfloat16_rn(acc / sum);
        } else if (dp.cluster_merge) {
            // to the CTA that finishes this row; a split without keys sends a log-sum of -inf
            const uint32_t dst = cluster_map(tc_smem(recv + (split * slots + m / csize) * L::RECV_ROW), m % csize);
            st_cluster_f32(dst + 4 * e, empty ? 0.f : acc / sum);
            if (e == 0) st_cluster_f32(dst + 4 * D, empty ? -INFINITY : mstar + log2f(sum));
        } else {
            const int64_t at = (((int64_t)ti * p.nkv + kvh) * dp.num_splits + split) * 16 + m;
            dp.part_o[at * D + e] = empty ? 0.f : acc / sum;
            if (e == 0) dp.part_lse[at] = empty ? -INFINITY : mstar + log2f(sum);
        }
    }
    if (dp.cluster_merge) {
        cg::this_cluster().sync();                               // all partial rows have arrived
        for (int idx = threadIdx.x; idx < slots * D; idx += DF8_THREADS) {
            const int slot = idx / D, e = idx - slot * D;
            const int m = split + slot * csize;                  // the rows this CTA finishes: rank, rank + csize, ...
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
}

// The splits of a (tile, kv head) from scratch: one CTA per (tile, kv head, row of the tile), a thread an entry.
template <int D>
__global__ void attention_decode_f8_merge_kernel(const DecodeF8Params dp) {
    pdl_wait();
    pdl_trigger();
    const F8AttnParams& p = dp.a;
    const int kvh = blockIdx.x, m = blockIdx.y, ti = blockIdx.z, e = threadIdx.x;
    const int r = p.tiles[2 * ti], q0 = p.tiles[2 * ti + 1], rep = p.nq / p.nkv;
    const int tok = p.row_start[r] + q0 + m / rep;
    if (tok >= p.row_start[r + 1]) return;
    const int64_t at0 = ((int64_t)ti * p.nkv + kvh) * dp.num_splits * 16 + m;
    float mstar = -INFINITY;
    for (int s = 0; s < dp.num_splits; ++s) mstar = fmaxf(mstar, dp.part_lse[at0 + 16 * s]);
    float sum = 0.f, acc = 0.f;
    for (int s = 0; s < dp.num_splits; ++s) {
        const float lse = dp.part_lse[at0 + 16 * s];
        const float f = lse == -INFINITY ? 0.f : exp2f(lse - mstar);
        sum += f;
        acc += f * dp.part_o[(at0 + 16 * s) * D + e];
    }
    p.out[((int64_t)tok * p.nq + kvh * rep + m % rep) * D + e] = __float2bfloat16_rn(acc / sum);
}

// What this kernel takes.
extern "C" int acorn_attention_decode_f8_supported(int nq, int nkv, int d, int P) {
    return nkv > 0 && nq % nkv == 0 && nq / nkv <= 16 && (d == 64 || d == 128) && P >= 8 && P <= 4096 && (P & (P - 1)) == 0;
}

// Whether this many splits are merged inside the kernel (by a cluster, without scratch).
extern "C" int acorn_attention_decode_f8_merges(int num_splits) { return num_splits <= 8 || num_splits == DF8_CLUSTER_MAX; }

// Codes [rows, D bytes], boxes of box_rows rows, swizzled over rows of D bytes.
static int make_map_codes(CUtensorMap* map, const void* base, int64_t rows, int d, int box_rows) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr || rows > 0x7fffffff) return ACORN_ERR_UNSUPPORTED;
    const cuuint64_t dims[2] = {(cuuint64_t)d, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)d};
    const cuuint32_t box[2] = {(cuuint32_t)d, (cuuint32_t)box_rows};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : 20000 + (int)r;
}

template <int D>
static int launch_decode_f8(const DecodeF8Params& dp, int64_t num_pages, int n_tiles, cudaStream_t stream) {
    using L = DecodeF8<D>;
    const F8AttnParams& p = dp.a;
    CUtensorMap mk, mv;
    const int P = 1 << p.logP, box_rows = P < DF8_CHUNK ? P : DF8_CHUNK;
    int rc = make_map_codes(&mk, p.k_pages, num_pages * p.nkv * P, D, box_rows);
    if (rc) return rc;
    rc = make_map_codes(&mv, p.v_pages, num_pages * p.nkv * P, D, box_rows);
    if (rc) return rc;
    const int rows = dp.tile_tokens * (p.nq / p.nkv);
    const size_t recv = dp.cluster_merge ? (size_t)dp.num_splits * ((rows + dp.num_splits - 1) / dp.num_splits) * L::RECV_ROW * 4 : 0;
    const size_t smem = L::RECV + recv, smem_max = L::RECV + (size_t)32 * L::RECV_ROW * 4;
    static AcornPerDevice configured;
    if (!configured.seen()) {
        cudaError_t e = cudaFuncSetAttribute(attention_decode_f8_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_max);
        if (e != cudaSuccess) return (int)e;
        e = cudaFuncSetAttribute(attention_decode_f8_kernel<D>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return (int)e;
        configured.mark();
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.nkv, dp.num_splits, n_tiles);
    cfg.blockDim = dim3(DF8_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = dp.cluster_merge ? dp.num_splits : 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = acorn_pdl_enabled() ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, attention_decode_f8_kernel<D>, mk, mv, dp);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess || dp.num_splits == 1 || dp.cluster_merge) return (int)e;
    return acorn_launch(attention_decode_f8_merge_kernel<D>, dim3(p.nkv, rows, n_tiles), dim3(D), 0, stream, dp);
}

extern "C" int acorn_attention_decode_f8(const void* q, int64_t q_stride, void* out, const void* k_pages, const void* v_pages,
                                         const void* scales, int64_t num_pages, const int* block_table, const int* page_base,
                                         int table_stride, const int* row_start, const int* row_pos, const int* tiles, int n_tiles,
                                         int nq, int nkv, int d, int P, float scale, int window, int chunk, int keep,
                                         const float* sink, int num_splits, float* part_o, float* part_lse, cudaStream_t stream) {
    if (n_tiles <= 0) return 0;
    if (!acorn_attention_decode_f8_supported(nq, nkv, d, P) || n_tiles > 65535 || num_splits < 1 || num_splits > 65535 || q_stride % 8)
        return ACORN_ERR_UNSUPPORTED;
    DecodeF8Params dp;
    F8AttnParams& p = dp.a;
    p.q = (const bf16*)q; p.q_stride = q_stride; p.out = (bf16*)out; p.k_pages = (const uint8_t*)k_pages;
    p.v_pages = (const uint8_t*)v_pages; p.scales = (const uint8_t*)scales; p.block_table = block_table; p.page_base = page_base;
    p.row_start = row_start; p.row_pos = row_pos; p.tiles = tiles; p.sink = sink; p.table_stride = table_stride;
    p.nq = nq; p.nkv = nkv; p.mask = {window, chunk, keep}; p.scale_log2 = scale * 1.4426950408889634f;
    p.logP = acorn_log2_exact_tc(P);
    dp.tile_tokens = 16 / (nq / nkv);
    dp.num_splits = num_splits;
    dp.cluster_merge = num_splits > 1 && acorn_attention_decode_f8_merges(num_splits);
    dp.part_o = part_o; dp.part_lse = part_lse;
    if (num_splits > 1 && !dp.cluster_merge && (part_o == nullptr || part_lse == nullptr)) return ACORN_ERR_UNSUPPORTED;
    return d == 128 ? launch_decode_f8<128>(dp, num_pages, n_tiles, stream) : launch_decode_f8<64>(dp, num_pages, n_tiles, stream);
}

extern "C" int acorn_attention_decode_f8_error() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_attn_dec_f8_error, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_attn_dec_f8_error, &zero, sizeof(int));
    return v;
}

ACORN_ERROR_WORD_SETTER(acorn_attention_decode_f8_set_error_word)
