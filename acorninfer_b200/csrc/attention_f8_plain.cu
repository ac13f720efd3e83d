// Attention over the pages of the 8-bit cache (f8_cache.cuh) for any head size that is a multiple of 8, any page size and any
// number of query heads per kv head: what the kernels for head sizes 64 and 128 do not take.
//
// One CTA per (token, query head): its four warps take every fourth run of 32 keys, a lane a key, so that a score is one
// lane's sum over the head and the softmax statistics of 32 keys are warp reductions; then a lane takes every 32nd entry of
// the values, the weights handed round by shuffles.  Running maximum, sum and output stay in float32; the warps are
// merged through shared memory.  Reads are not coalesced (a lane walks its own key row): right everywhere, fast nowhere.
#include "f8_cache.cuh"

#define F8P_THREADS 128
#define F8P_MAX_D 256

__global__ void __launch_bounds__(F8P_THREADS) attention_f8_plain_kernel(const F8AttnParams p, int d, int tile_tokens) {
    __shared__ float sq[F8P_MAX_D];
    __shared__ float so[4][F8P_MAX_D];
    __shared__ float sm[4], sl[4];
    pdl_wait();
    pdl_trigger();
    const int tile = blockIdx.x / tile_tokens, j = blockIdx.x % tile_tokens, head = blockIdx.y;
    const int r = p.tiles[2 * tile], i0 = p.tiles[2 * tile + 1] + j;
    const int t = p.row_start[r] + i0;
    if (t >= p.row_start[r + 1]) return;
    const int pos = p.row_pos[r] + i0, kvh = head / (p.nq / p.nkv);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < d; i += F8P_THREADS) sq[i] = to_float(p.q[(int64_t)t * p.q_stride + (int64_t)head * d + i]);
    __syncthreads();
    const int lo = mask_lo(p.mask, pos), vlo = mask_vlo(p.mask, lo), hi = pos + 1;
    const int* table = p.block_table + (int64_t)r * p.table_stride - p.page_base[r];
    const int pmask = (1 << p.logP) - 1;
    float m = -INFINITY, sum = 0.f, o[F8P_MAX_D / 32];
#pragma unroll
    for (int i = 0; i < F8P_MAX_D / 32; ++i) o[i] = 0.f;
    for (int v0 = vlo + 32 * warp; v0 < hi; v0 += 128) {
        const int v = v0 + lane;
        int64_t slot = 0;
        float s = -INFINITY, vs = 0.f;
        if (v < hi) {
            const int key = mask_key(v, vlo, lo);
            slot = (((int64_t)table[key >> p.logP] * p.nkv + kvh) << p.logP) + (key & pmask);
            const uint32_t* row = reinterpret_cast<const uint32_t*>(p.k_pages + slot * d);
            float acc = 0.f;
            for (int i = 0; i < d / 4; ++i) {
                const uint32_t c = row[i];
                const float2 a = f8_codes2(c), b = f8_codes2(c >> 16);
                acc = fmaf(a.x, sq[4 * i], fmaf(a.y, sq[4 * i + 1], fmaf(b.x, sq[4 * i + 2], fmaf(b.y, sq[4 * i + 3], acc))));
            }
            vs = f8_scale(p.scales[2 * slot + 1]);
            s = acc * p.scale_log2 * f8_scale(p.scales[2 * slot]);
            if (isnan(vs)) { s = vs; vs = 0.f; }              // a value row that is no number makes the query's whole result NaN
        }
        const float mn = fmaxf(m, warp_max(s));
        const float corr = m == -INFINITY ? 0.f : exp2f(m - mn);
        const float w = v < hi ? exp2f(s - mn) : 0.f;
        m = mn;
        sum = sum * corr + warp_sum(w);
        const float wv = w * vs;
#pragma unroll
        for (int i = 0; i < F8P_MAX_D / 32; ++i) o[i] *= corr;
        for (int k = 0; k < 32 && v0 + k < hi; ++k) {
            const float wk = __shfl_sync(0xffffffffu, wv, k);
            const int64_t at = __shfl_sync(0xffffffffu, slot, k) * d;
#pragma unroll
            for (int i = 0; i < F8P_MAX_D / 32; ++i)
                if (32 * i + lane < d) o[i] = fmaf(wk, f8_codes2(p.v_pages[at + 32 * i + lane]).x, o[i]);
        }
    }
    if (lane == 0) { sm[warp] = m; sl[warp] = sum; }
#pragma unroll
    for (int i = 0; i < F8P_MAX_D / 32; ++i)
        if (32 * i + lane < d) so[warp][32 * i + lane] = o[i];
    __syncthreads();
    const float sink = p.sink ? p.sink[head] * 1.4426950408889634f : -INFINITY;
    const float top = fmaxf(fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), sink);
    float total = exp2f(sink - top), f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        // a warp without keys adds nothing; one whose keys are all NaN has no maximum, but a sum that is NaN
        f[w] = sm[w] == -INFINITY && sl[w] == 0.f ? 0.f : exp2f(sm[w] - top);
        total += f[w] == 0.f && !isnan(sl[w]) ? 0.f : f[w] * sl[w];
    }
    for (int i = threadIdx.x; i < d; i += F8P_THREADS) {
        const float acc = f[0] * so[0][i] + f[1] * so[1][i] + f[2] * so[2][i] + f[3] * so[3][i];
        p.out[((int64_t)t * p.nq + head) * d + i] = __float2bfloat16_rn(acc / total);
    }
}

extern "C" int acorn_attention_f8_plain(const void* q, int64_t q_stride, void* out, const void* k_pages, const void* v_pages,
                                        const void* scales, const int* block_table, const int* page_base, int table_stride,
                                        const int* row_start, const int* row_pos, const int* tiles, int n_tiles,
                                        int tile_tokens, int nq, int nkv, int d, int P, float scale, int window, int chunk,
                                        int keep, const float* sink, cudaStream_t stream) {
    if (n_tiles <= 0) return 0;
    if (d < 8 || d % 8 || d > F8P_MAX_D || P < 1 || (P & (P - 1)) || nkv < 1 || nq % nkv || nq > 65535 || tile_tokens < 1 ||
        (int64_t)n_tiles * tile_tokens > 0x7fffffff)
        return ACORN_ERR_UNSUPPORTED;
    F8AttnParams p;
    p.q = (const bf16*)q; p.q_stride = q_stride; p.out = (bf16*)out; p.k_pages = (const uint8_t*)k_pages;
    p.v_pages = (const uint8_t*)v_pages; p.scales = (const uint8_t*)scales; p.block_table = block_table; p.page_base = page_base;
    p.row_start = row_start; p.row_pos = row_pos; p.tiles = tiles; p.sink = sink; p.table_stride = table_stride;
    p.nq = nq; p.nkv = nkv; p.mask = {window, chunk, keep}; p.scale_log2 = scale * 1.4426950408889634f;
    p.logP = 0;
    while ((1 << p.logP) < P) ++p.logP;
    return acorn_launch(attention_f8_plain_kernel, dim3((unsigned)(n_tiles * tile_tokens), nq), dim3(F8P_THREADS), 0, stream, p, d,
                        tile_tokens);
}
