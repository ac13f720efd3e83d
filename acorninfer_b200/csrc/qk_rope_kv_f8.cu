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
// a lane takes eight neighbouring entries of a head (16 bytes in; 16 or 8 out), LPH lanes a head, so that the sum of squares,
// the largest magnitude and the other half of a rotated pair are shuffles among them.  The angle is formed and brought to
// [-pi, pi] in 64 bits: in 32 its error is 2^-24 of the angle itself, 0.008 radians at position 131,072, against 2^-9 of a
// rounding to bfloat16.
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
    int table_stride, nq, nkv, d, rot, interleaved, P;
    float eps, magnitude;
};

__device__ __forceinline__ void kvf8_unpack(const uint4& raw, float (&x)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

template <int LPH>
__global__ void __launch_bounds__(KVF8_THREADS) qk_rope_kv_f8_kernel(const KvF8Params p) {
    extern __shared__ float2 turn[];                          // cos and sin of the token's angles
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x;
    const int pos = p.positions[t];
    const int half = p.rot >> 1;
    for (int j = threadIdx.x; j < half; j += KVF8_THREADS) {
        const double a = (double)pos * (double)p.inv_freq[j];
        const double r = fma(-rint(a * 0.15915494309189535), 6.283185307179586, a);
        float s, c;
        sincosf((float)r, &s, &c);
        turn[j] = make_float2(c * p.magnitude, s * p.magnitude);
    }
    __syncthreads();
    const int heads = p.nq + 2 * p.nkv;
    const int l = threadIdx.x & (LPH - 1);
    const bool on = 8 * l < p.d;                              // lanes beyond a head whose size is no power of two
    const int per_pass = KVF8_THREADS / LPH * gridDim.y;
    for (int h0 = blockIdx.y * (KVF8_THREADS / LPH); h0 < heads; h0 += per_pass) {       // the same trips for all lanes of a warp
        const int h = h0 + threadIdx.x / LPH;
        const bool live = on && h < heads;
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (live) kvf8_unpack(*reinterpret_cast<const uint4*>(p.qkv + (int64_t)t * p.ld + (int64_t)h * p.d + 8 * l), x);
        if (p.bias && live) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] += p.bias[h * p.d + 8 * l + i];
        }
        const bool is_v = h >= p.nq + p.nkv;
        const float* w = is_v ? nullptr : h < p.nq ? p.q_w : p.k_w;
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (w && live) {
            const float inv = rsqrtf(ss / (float)p.d + p.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * w[8 * l + i];
        }
        if (p.interleaved) {
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
            const int step = half >> 3;
            const bool first = l < step, second = !first && l < 2 * step;
            const int from = (threadIdx.x & 31 & ~(LPH - 1)) + (first ? l + step : second ? l - step : l);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], from);
            if (!is_v && (first || second) && live) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 cs = turn[8 * (first ? l : l - step) + i];
                    x[i] = x[i] * cs.x + (first ? -y[i] : y[i]) * cs.y;
                }
            }
        }
        float most = 0.f;
        bool finite = true;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            most = fmaxf(most, fabsf(x[i]));
            finite = finite && fabsf(x[i]) <= 3.402823466e38f;
        }
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) {
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            finite = __shfl_xor_sync(0xffffffffu, (int)finite, o) && finite;
        }
        if (!live) continue;
        if (h < p.nq) {
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                v[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
            *reinterpret_cast<uint4*>(p.q_out + (int64_t)t * p.ld_q + (int64_t)h * p.d + 8 * l) = make_uint4(v[0], v[1], v[2], v[3]);
            continue;
        }
        const int r = p.token_row[t], kvh = (h - p.nq) % p.nkv;
        const int page = p.block_table[(int64_t)r * p.table_stride + (pos / p.P - p.page_base[r])];
        const int64_t slot = ((int64_t)page * p.nkv + kvh) * p.P + pos % p.P;
        const int e = f8_row_exponent(most);
        // at the largest exponent a code above 240 would stand for more than the largest float
        const float inv = finite ? f8_pow2(-e) : 0.f, limit = e == F8_MAX_EXP ? 240.f : 448.f;
        uint32_t c[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float z[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) z[k] = finite ? fminf(fmaxf(x[4 * i + k] * inv, -limit), limit) : 0.f;
            c[i] = f8_pack2(z[0], z[1]) | f8_pack2(z[2], z[3]) << 16;
        }
        *reinterpret_cast<uint2*>((is_v ? p.v_pages : p.k_pages) + slot * p.d + 8 * l) = make_uint2(c[0], c[1]);
        if (l == 0) p.scales[2 * slot + (is_v ? 1 : 0)] = (uint8_t)(finite ? e + 127 : F8_NAN_BYTE);
    }
}

extern "C" int acorn_qk_rope_kv_f8(const void* qkv, int64_t ld, const float* q_w, const float* k_w, const float* bias,
                                   const float* inv_freq, const int* positions, const int* token_row, const int* block_table,
                                   const int* page_base, int table_stride, void* k_pages, void* v_pages, void* scales,
                                   void* q_out, int64_t ld_q, int tokens, int nq, int nkv, int d, int rot, int interleaved,
                                   int P, float eps, float magnitude, cudaStream_t stream) {
    if (tokens <= 0) return 0;
    if (d < 8 || d % 8 || d > 256 || rot < 0 || rot > d || rot % (interleaved ? 2 : 16) || P < 1 || nq < 1 || nkv < 1 ||
        ld % 8 || ld_q % 8)
        return ACORN_ERR_UNSUPPORTED;
    KvF8Params p;
    p.qkv = (const bf16*)qkv; p.ld = ld; p.q_w = q_w; p.k_w = k_w; p.bias = bias; p.inv_freq = inv_freq; p.positions = positions;
    p.token_row = token_row; p.block_table = block_table; p.page_base = page_base; p.k_pages = (uint8_t*)k_pages;
    p.v_pages = (uint8_t*)v_pages; p.scales = (uint8_t*)scales; p.q_out = (bf16*)q_out; p.ld_q = ld_q; p.table_stride = table_stride;
    p.nq = nq; p.nkv = nkv; p.d = d; p.rot = rot; p.interleaved = interleaved; p.P = P; p.eps = eps; p.magnitude = magnitude;
    int lph = 1;
    while (8 * lph < d) lph *= 2;
    const int passes = (nq + 2 * nkv + KVF8_THREADS / lph - 1) / (KVF8_THREADS / lph);
    const dim3 grid(tokens, tokens < 2 * acorn_sms() ? passes : 1);
    const size_t smem = (size_t)(rot / 2) * sizeof(float2);
    switch (lph) {
        case 1: return acorn_launch(qk_rope_kv_f8_kernel<1>, grid, dim3(KVF8_THREADS), smem, stream, p);
        case 2: return acorn_launch(qk_rope_kv_f8_kernel<2>, grid, dim3(KVF8_THREADS), smem, stream, p);
        case 4: return acorn_launch(qk_rope_kv_f8_kernel<4>, grid, dim3(KVF8_THREADS), smem, stream, p);
        case 8: return acorn_launch(qk_rope_kv_f8_kernel<8>, grid, dim3(KVF8_THREADS), smem, stream, p);
        case 16: return acorn_launch(qk_rope_kv_f8_kernel<16>, grid, dim3(KVF8_THREADS), smem, stream, p);
        default: return acorn_launch(qk_rope_kv_f8_kernel<32>, grid, dim3(KVF8_THREADS), smem, stream, p);
    }
}
