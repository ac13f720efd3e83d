// Per-head q/k RMSNorm + rotary position encoding + write of K and V into the pages of the 8-bit cache (f8_cache.cuh).
//
// qkv is the projection output [tokens, ld]: nq query heads, nkv key heads, nkv value heads of d entries each.  For every
// token and head, in float32:
//   all heads:   x <- x + bias                                       (if biases are given)
//   q, k heads:  x <- x * rsqrt(mean(x^2) + eps) * w                  (if a norm weight is given)
//                the first `rot` entries are rotated by the angle pos * inv_freq[j], cos and sin times `magnitude`, in pairs
//                (x[j], x[j + rot/2]) or (x[2j], x[2j + 1])
//   q heads are rounded to bfloat16 into q_out; k and v heads become e4m3 codes and an exponent, straight from float32.
//
// A CTA takes one token, or a share of its heads where tokens are few: the token's angles are made once, in shared memory, and
// a lane takes eight entries of a head (16 bytes in; 16 or 8 out), LPH lanes a head, so that the sum of squares and the
// largest magnitude are shuffles among them.  Heads rotated whole in pairs (j, j + d/2) give a lane four entries of each half, so
// that it holds whole pairs (PAIRED); otherwise the eight are neighbours, and the other half of a pair is a shuffle more.
// What bounds it: its instructions, not its bytes; so only the key and value heads look for their largest magnitude, by a
// maximum that hands NaN on, which tells infinities and NaN as well.  Without pages the queries alone are made (a layer that reads
// another one's cache), with the very same angles.
#include "f8_cache.cuh"

#define KVF8_THREADS 256

struct KvF8Params {
    const bf16* qkv;
    int64_t ld;
    const float* q_w;
    const float* k_w;
    const float* bias;        // [(nq + 2 nkv) d] or null
    const float* inv_freq;    // [rot / 2]
    const int* positions;
    const int* token_row;
    const int* block_table;
    const int* page_base;
    uint8_t* k_pages;
    uint8_t* v_pages;
    uint8_t* scales;
    bf16* q_out;
    int64_t ld_q;
    int tokens, table_stride, nq, nkv, d, rot, interleaved, logP;
    float inv_d, eps, magnitude;
};

__device__ __forceinline__ void kvf8_unpack(const uint4& raw, float (&x)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ uint2 kvf8_pack4(float a, float b, float c, float d) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Eight entries times 2^-e as codes.  At the largest exponent a code above 240 would stand for more than the largest float.
__device__ __forceinline__ uint2 kvf8_codes(const float (&x)[8], int e) {
    float z[8];
    const float inv = f8_pow2(-e);
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = x[i] * inv;
    if (e == F8_MAX_EXP) {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = fminf(fmaxf(z[i], -240.f), 240.f);
    }
    return make_uint2(f8_pack2(z[0], z[1]) | f8_pack2(z[2], z[3]) << 16, f8_pack2(z[4], z[5]) | f8_pack2(z[6], z[7]) << 16);
}

template <int LPH, bool PAIRED, bool WRITE>
__global__ void __launch_bounds__(KVF8_THREADS, 8) qk_rope_kv_f8_kernel(const KvF8Params p) {
    extern __shared__ __align__(16) float2 turn[];            // cos and sin of the token's angles
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x;
    const int pos = p.positions[t], r = p.token_row[t];
    const int half = p.rot >> 1;
    const int heads = WRITE ? p.nq + 2 * p.nkv : p.nq;
    const int l = threadIdx.x & (LPH - 1);
    const bool on = 8 * l < p.d;                              // lanes beyond a head whose size is no power of two
    // this lane's entries: at0 .. at0 + 3 and at1 .. at1 + 3
    const int at0 = PAIRED ? 4 * l : 8 * l, at1 = PAIRED ? (p.d >> 1) + 4 * l : 8 * l + 4;
    const bf16* row = p.qkv + (int64_t)t * p.ld;
    auto fetch = [&](int h) {
        if (!on || h >= heads) return make_uint4(0u, 0u, 0u, 0u);
        const bf16* src = row + h * p.d;
        const uint2 a = *reinterpret_cast<const uint2*>(src + at0), b = *reinterpret_cast<const uint2*>(src + at1);
        return make_uint4(a.x, a.y, b.x, b.y);
    };
    const int in_pass = threadIdx.x / LPH, per_cta = blockDim.x / LPH, per_pass = per_cta * gridDim.y;
    int h0 = blockIdx.y * per_cta;
    uint4 raw = fetch(h0 + in_pass);                          // on its way while the angles are made
    const int page = WRITE ? p.block_table[(int64_t)r * p.table_stride + ((pos >> p.logP) - p.page_base[r])] : 0;
    for (int j = threadIdx.x; j < half; j += blockDim.x) {
        const float2 cs = f8_turn(pos, p.inv_freq[j]);
        turn[j] = make_float2(cs.x * p.magnitude, cs.y * p.magnitude);
    }
    __syncthreads();
    const int64_t slot0 = (((int64_t)page * p.nkv) << p.logP) + (pos & ((1 << p.logP) - 1));
    for (; h0 < heads; h0 += per_pass) {                      // the same trips for all lanes of a warp
        const int h = h0 + in_pass;
        const bool live = on && h < heads;
        float x[8];
        kvf8_unpack(raw, x);
        raw = fetch(h + per_pass);
        if (p.bias && live) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] += p.bias[h * p.d + (i < 4 ? at0 + i : at1 + i - 4)];
        }
        const bool is_v = h >= p.nq + p.nkv;
        const float* w = is_v ? nullptr : h < p.nq ? p.q_w : p.k_w;
        if (p.q_w || p.k_w) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const bool large = w && ss == INFINITY;
            if (__any_sync(0xffffffffu, large)) {             // rare: the same for a row brought down
                if (large) {
                    ss = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) { x[i] *= F8_NORM_DOWN; ss = fmaf(x[i], x[i], ss); }
                }
                float all = ss;
#pragma unroll
                for (int o = LPH / 2; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
                if (large) ss = all;
            }
            if (w && live) {
                const float inv = f8_inverse_root(fmaf(ss, p.inv_d, large ? 0.f : p.eps));
                const float4 wa = *reinterpret_cast<const float4*>(w + at0), wb = *reinterpret_cast<const float4*>(w + at1);
                x[0] *= inv * wa.x; x[1] *= inv * wa.y; x[2] *= inv * wa.z; x[3] *= inv * wa.w;
                x[4] *= inv * wb.x; x[5] *= inv * wb.y; x[6] *= inv * wb.z; x[7] *= inv * wb.w;
            }
        }
        if constexpr (PAIRED) {
            if (!is_v && live) {
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float4 cs = *reinterpret_cast<const float4*>(turn + at0 + i);
                    const float a0 = x[i], b0 = x[4 + i], a1 = x[i + 1], b1 = x[5 + i];
                    x[i] = a0 * cs.x - b0 * cs.y; x[4 + i] = b0 * cs.x + a0 * cs.y;
                    x[i + 1] = a1 * cs.z - b1 * cs.w; x[5 + i] = b1 * cs.z + a1 * cs.w;
                }
            }
        } else if (p.interleaved) {
            if (live && !is_v && 8 * l < p.rot) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const int j = 4 * l + (i >> 1);
                    if (j < half) {
                        const float2 cs = turn[j];
                        const float a = x[i], b = x[i + 1];
                        x[i] = a * cs.x - b * cs.y;
                        x[i + 1] = b * cs.x + a * cs.y;
                    }
                }
            }
        } else if (half > 0) {                                // half is a multiple of 8: the partner is another lane's entry
            const int away = half >> 3;
            const bool first = l < away, second = !first && l < 2 * away;
            const int from = (threadIdx.x & 31 & ~(LPH - 1)) + (first ? l + away : second ? l - away : l);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], from);
            if (!is_v && (first || second) && live) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 cs = turn[8 * (first ? l : l - away) + i];
                    x[i] = x[i] * cs.x + (first ? -y[i] : y[i]) * cs.y;
                }
            }
        }
        if (__all_sync(0xffffffffu, h < p.nq)) {              // queries throughout the warp
            if (live) {
                bf16* dst = p.q_out + (int64_t)t * p.ld_q + (int64_t)h * p.d;
                *reinterpret_cast<uint2*>(dst + at0) = kvf8_pack4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<uint2*>(dst + at1) = kvf8_pack4(x[4], x[5], x[6], x[7]);
            }
            continue;
        }
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max_nan(most, fabsf(x[i]));
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
        if (!live) continue;
        if (h < p.nq) {
            bf16* dst = p.q_out + (int64_t)t * p.ld_q + (int64_t)h * p.d;
            *reinterpret_cast<uint2*>(dst + at0) = kvf8_pack4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<uint2*>(dst + at1) = kvf8_pack4(x[4], x[5], x[6], x[7]);
            continue;
        }
        const int64_t slot = slot0 + ((h - p.nq - (is_v ? p.nkv : 0)) << p.logP);
        const bool finite = most <= 3.402823466e38f;
        const int e = f8_row_exponent(most);
        const uint2 c = finite ? kvf8_codes(x, e) : make_uint2(0u, 0u);
        uint8_t* dst = (is_v ? p.v_pages : p.k_pages) + slot * p.d;
        if constexpr (PAIRED) {
            *reinterpret_cast<uint32_t*>(dst + at0) = c.x;
            *reinterpret_cast<uint32_t*>(dst + at1) = c.y;
        } else {
            *reinterpret_cast<uint2*>(dst + at0) = c;
        }
        if (l == 0) p.scales[2 * slot + (is_v ? 1 : 0)] = (uint8_t)(finite ? e + 127 : F8_NAN_BYTE);
    }
}

template <int LPH, bool PAIRED, bool WRITE>
static int launch_kv_f8(const KvF8Params& p, cudaStream_t stream) {
    // as few passes as 256 threads need, and as many threads as those passes leave no idle ones; few tokens: a CTA a pass
    const int lanes = (WRITE ? p.nq + 2 * p.nkv : p.nq) * LPH, passes = (lanes + KVF8_THREADS - 1) / KVF8_THREADS;
    const int threads = ((lanes + passes - 1) / passes + 31) / 32 * 32;
    return acorn_launch(qk_rope_kv_f8_kernel<LPH, PAIRED, WRITE>, dim3(p.tokens, p.tokens < 2 * acorn_sms() ? passes : 1), dim3(threads),
                        (size_t)(p.rot / 2) * sizeof(float2), stream, p);
}

template <int LPH>
static int launch_kv_f8(const KvF8Params& p, cudaStream_t stream) {
    const bool paired = p.rot == p.d && !p.interleaved;
    if (p.k_pages == nullptr) return paired ? launch_kv_f8<LPH, true, false>(p, stream) : launch_kv_f8<LPH, false, false>(p, stream);
    return paired ? launch_kv_f8<LPH, true, true>(p, stream) : launch_kv_f8<LPH, false, true>(p, stream);
}

extern "C" int acorn_qk_rope_kv_f8(const void* qkv, int64_t ld, const float* q_w, const float* k_w, const float* bias,
                                   const float* inv_freq, const int* positions, const int* token_row, const int* block_table,
                                   const int* page_base, int table_stride, void* k_pages, void* v_pages, void* scales,
                                   void* q_out, int64_t ld_q, int tokens, int nq, int nkv, int d, int rot, int interleaved,
                                   int P, float eps, float magnitude, cudaStream_t stream) {
    if (tokens <= 0) return 0;
    if ((k_pages == nullptr) != (v_pages == nullptr) || (k_pages == nullptr) != (scales == nullptr)) return ACORN_ERR_UNSUPPORTED;
    if (d < 8 || d % 8 || d > 256 || rot < 0 || rot > d || rot % (interleaved ? 2 : 16) || P < 1 || (P & (P - 1)) || nq < 1 || nkv < 1 ||
        ld % 8 || ld_q % 8)
        return ACORN_ERR_UNSUPPORTED;
    KvF8Params p;
    p.qkv = (const bf16*)qkv; p.ld = ld; p.q_w = q_w; p.k_w = k_w; p.bias = bias; p.inv_freq = inv_freq; p.positions = positions;
    p.token_row = token_row; p.block_table = block_table; p.page_base = page_base; p.k_pages = (uint8_t*)k_pages;
    p.v_pages = (uint8_t*)v_pages; p.scales = (uint8_t*)scales; p.q_out = (bf16*)q_out; p.ld_q = ld_q; p.table_stride = table_stride;
    p.tokens = tokens; p.nq = nq; p.nkv = nkv; p.d = d; p.rot = rot; p.interleaved = interleaved; p.eps = eps; p.inv_d = 1.f / (float)d;
    p.logP = 0;
    while ((1 << p.logP) < P) ++p.logP;
    p.magnitude = magnitude;
    int lph = 1;
    while (8 * lph < d) lph *= 2;
    switch (lph) {
        case 1: return launch_kv_f8<1>(p, stream);
        case 2: return launch_kv_f8<2>(p, stream);
        case 4: return launch_kv_f8<4>(p, stream);
        case 8: return launch_kv_f8<8>(p, stream);
        case 16: return launch_kv_f8<16>(p, stream);
        default: return launch_kv_f8<32>(p, stream);
    }
}
