// kvm_qkrope.cu -- kvm_qk_norm_rope: RMS norm of every query and key head and
// the NeoX rotation, one pass over the values.
//
//   y = x * rsqrt(mean(x^2) + eps) * w;   (y_i, y_{i+h}) -> (y_i c - y_{i+h} s, y_{i+h} c + y_i s)
//
// h = n_rot / 2, (c, s) = cos, sin of pos * freq_i.  The angle is a product of
// an integer and an F32 value, exact in F64 up to 2^29 and within 2^-53 beyond;
// it is reduced by whole turns in F64 (a far position would lose every digit in
// F32) and only the remainder goes to F32.  Norm, rotation and sums
// are F32 and each value is rounded once, at the store.
//
// Bound by HBM: every value is read and written once.  A thread owns the chunk
// pair that a rotation mixes (8 values and their partners n_rot/2 further on), so
// the rotation needs no exchange and the norm only a reduction over the head's
// head_dim/16 neighbouring threads.  A CTA takes one to four tokens at a time, all
// heads: its threads first issue the loads of two heads each (four vectors; 64
// registers and so four CTAs an SM, which beat eight vectors at three), then form
// the tokens' cos / sin once for all heads, in shared memory, while those loads
// are under way.  The query weights stay in registers across the tokens.
//
// 8192 tokens of 24 + 4 heads of 256, BF16, all rotated: 51 us for 235 MB = 4.6 TB/s
// (a copy 36 us): issue slots 59 % busy, norm and rotation cost 18 instructions a
// pair of values.  64 tokens: 4.2 us, launch and two dependent loads.
#include <cuda_bf16.h>

#include <algorithm>

#include "kvm_layer.cuh"

namespace kvm {
namespace {

constexpr int kRopeThreads = 256;
constexpr uint32_t kRopeMaxDim = 512;

struct RopeTensor {
    const uint8_t *src;
    uint8_t *dst;
    const float *weight;
    uint64_t s_dim, s_head, s_tok, d_dim, d_head, d_tok;
    uint32_t heads;
};

struct RopeArgs {
    RopeTensor q, k;
    const float *freqs;
    const int32_t *pos;
    float eps;
    uint32_t head_dim, n_rot, lanes;   // lanes: threads a head, a power of two >= head_dim / 16
    uint32_t n, tokens;                // rows; rows a CTA takes at a time
    float inv_dim;                     // 1 / head_dim
};

// Eight values as they lie in memory (16-bit types: four words).
template <int TYPE>
struct Raw8 {
    uint32_t w[TYPE == KVM_TYPE_F32 ? 8 : 4];
};

template <int TYPE, bool VEC>
__device__ __forceinline__ void load8(const uint8_t *p, uint64_t nb_dim, Raw8<TYPE> &r) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (TYPE == KVM_TYPE_F32 ? 2 : 1); ++i) {
            const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
            r.w[4 * i] = v.x; r.w[4 * i + 1] = v.y; r.w[4 * i + 2] = v.z; r.w[4 * i + 3] = v.w;
        }
    } else if constexpr (TYPE == KVM_TYPE_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.w[i] = *reinterpret_cast<const uint32_t *>(p + i * nb_dim);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r.w[i] = *reinterpret_cast<const uint16_t *>(p + 2 * i * nb_dim) |
                     static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(p + (2 * i + 1) * nb_dim)) << 16;
    }
}

template <int TYPE>
__device__ __forceinline__ void widen8(const Raw8<TYPE> &r, float2 (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (TYPE == KVM_TYPE_F32) x[i] = make_float2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
        else if constexpr (TYPE == KVM_TYPE_F16) x[i] = __half22float2(*reinterpret_cast<const __half2 *>(&r.w[i]));
        else x[i] = make_float2(__uint_as_float(r.w[i] << 16), __uint_as_float(r.w[i] & 0xffff0000u));
    }
}

template <int TYPE>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (TYPE == KVM_TYPE_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

template <int TYPE, bool VEC>
__device__ __forceinline__ void store8(uint8_t *p, uint64_t nb_dim, const float2 (&x)[4]) {
    if constexpr (VEC && TYPE == KVM_TYPE_F32) {
        *reinterpret_cast<float4 *>(p) = make_float4(x[0].x, x[0].y, x[1].x, x[1].y);
        *reinterpret_cast<float4 *>(p + 16) = make_float4(x[2].x, x[2].y, x[3].x, x[3].y);
    } else if constexpr (VEC) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack2<TYPE>(x[0].x, x[0].y), pack2<TYPE>(x[1].x, x[1].y),
                                                   pack2<TYPE>(x[2].x, x[2].y), pack2<TYPE>(x[3].x, x[3].y));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint8_t *e = p + i * nb_dim;
            const float v = i & 1 ? x[i / 2].y : x[i / 2].x;
            if constexpr (TYPE == KVM_TYPE_F32) *reinterpret_cast<float *>(e) = v;
            else *reinterpret_cast<uint16_t *>(e) = static_cast<uint16_t>(pack2<TYPE>(v, 0.0f) & 0xffffu);
        }
    }
}

template <bool VEC>
__device__ __forceinline__ void load_weights(const float *w, uint32_t e, float2 (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (!w) x[i] = make_float2(1.0f, 1.0f);
        else if constexpr (VEC) x[i] = *reinterpret_cast<const float2 *>(w + e + 2 * i);
        else x[i] = make_float2(w[e + 2 * i], w[e + 2 * i + 1]);
    }
}

// Byte offset of a head of a row.  Vector accesses come with strides below 2^32
// (two wide multiply-adds); others take any.
template <bool VEC>
__device__ __forceinline__ uint64_t head_offset(uint32_t tok, uint64_t s_tok, uint32_t h, uint64_t s_head) {
    if constexpr (VEC)
        return static_cast<uint64_t>(tok) * static_cast<uint32_t>(s_tok) + static_cast<uint64_t>(h) * static_cast<uint32_t>(s_head);
    else
        return tok * s_tok + h * s_head;
}

constexpr int kRopeTokens = 4;
// floats between two threads' 8 cos (then 8 sin) values: 16-byte reads of eight
// neighbouring threads fall into different banks
constexpr int kRopePitch = 12;

template <int TYPE, bool VEC>
__global__ void __launch_bounds__(kRopeThreads, 4) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
    constexpr int kBatch = TYPE == KVM_TYPE_F32 ? 1 : 2;      // heads of a thread in flight
    constexpr uint64_t kEs = TYPE == KVM_TYPE_F32 ? 4 : 2;
    __shared__ __align__(16) float cs[2][kRopeTokens][kRopeMaxDim / 16 * kRopePitch];
    const uint32_t half = a.n_rot / 2, pairs = a.n_rot / 16;
    const uint32_t p = threadIdx.x & (a.lanes - 1), grp = threadIdx.x / a.lanes, groups = kRopeThreads / a.lanes;
    const uint32_t heads = a.q.heads + a.k.heads;
    const uint32_t rounds = (heads + groups - 1) / groups;
    const bool in = p < a.head_dim / 16, rot = p < pairs;
    // the two chunks of 8 of this thread
    const uint32_t e0 = rot ? 8 * p : a.n_rot + 16 * (p - pairs), e1 = rot ? e0 + half : e0 + 8;
    float2 wq0[4], wq1[4];
    if (in) {
        load_weights<VEC>(a.q.weight, e0, wq0);
        load_weights<VEC>(a.q.weight, e1, wq1);
    }
    for (uint32_t tok0 = blockIdx.x * a.tokens; tok0 < a.n; tok0 += gridDim.x * a.tokens) {
        const uint32_t toks = min(a.tokens, a.n - tok0);
        // item: (token, round), this thread's head of it
        const uint32_t items = toks * rounds;
        bool ready = false;
        uint32_t tk_in = 0, rd_in = 0, tk = 0, rd = 0;      // (token, round) of the next load, of the next result
        for (uint32_t i0 = 0; i0 < items; i0 += kBatch) {
            Raw8<TYPE> r0[kBatch], r1[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const uint32_t h = rd_in * groups + grp;
                if (in && tk_in < toks && h < heads) {
                    const bool key = h >= a.q.heads;
                    const RopeTensor &t = key ? a.k : a.q;
                    const uint8_t *src = t.src + head_offset<VEC>(tok0 + tk_in, t.s_tok, key ? h - a.q.heads : h, t.s_head);
                    load8<TYPE, VEC>(src + e0 * (VEC ? kEs : t.s_dim), t.s_dim, r0[k]);
                    load8<TYPE, VEC>(src + e1 * (VEC ? kEs : t.s_dim), t.s_dim, r1[k]);
                }
                if (++rd_in == rounds) {
                    rd_in = 0;
                    ++tk_in;
                }
            }
            if (!ready) {
                for (uint32_t x = threadIdx.x; x < toks * half; x += kRopeThreads) {
                    const uint32_t of = x / half, i = x - of * half;
                    const double ang = static_cast<double>(a.pos[tok0 + of]) * static_cast<double>(a.freqs[i]);
                    // in half turns: 1 / pi to 106 bits, its F64 value and the remainder
                    const double turn = ang * 0.31830988618379067154;
                    const double rest = fma(ang, 0.31830988618379067154, -turn) + ang * -1.9678676675182486e-17;
                    const double near = turn - 2.0 * rint(0.5 * turn);
                    float sn, co;
                    sincospif(static_cast<float>(near + rest), &sn, &co);
                    const uint32_t at = (i / 8) * kRopePitch + (i & 7);
                    cs[0][of][at] = co;
                    cs[1][of][at] = sn;
                }
                __syncthreads();
                ready = true;
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const uint32_t h = rd * groups + grp, row = tk;
                if (row >= toks) break;            // alike in the whole CTA
                if (++rd == rounds) {
                    rd = 0;
                    ++tk;
                }
                const bool on = in && h < heads, key = h >= a.q.heads;
                float2 x0[4] = {}, x1[4] = {}, s2 = make_float2(0.0f, 0.0f);
                if (on) {
                    widen8<TYPE>(r0[k], x0);
                    widen8<TYPE>(r1[k], x1);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s2 = f2_fma_rn(x1[e], x1[e], f2_fma_rn(x0[e], x0[e], s2));
                float ss = s2.x + s2.y;
                for (uint32_t o = a.lanes / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (!on) continue;
                const float rs = rsqrtf(ss * a.inv_dim + a.eps);
                const float2 rs2 = make_float2(rs, rs);
                if (key) {                         // few heads: weights from the cache
                    float2 w0[4], w1[4];
                    load_weights<VEC>(a.k.weight, e0, w0);
                    load_weights<VEC>(a.k.weight, e1, w1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x0[e] = f2_mul_rn(x0[e], f2_mul_rn(rs2, w0[e]));
                        x1[e] = f2_mul_rn(x1[e], f2_mul_rn(rs2, w1[e]));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x0[e] = f2_mul_rn(x0[e], f2_mul_rn(rs2, wq0[e]));
                        x1[e] = f2_mul_rn(x1[e], f2_mul_rn(rs2, wq1[e]));
                    }
                }
                if (rot) {
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const float4 co = *reinterpret_cast<const float4 *>(&cs[0][row][p * kRopePitch + 2 * e]);
                        const float4 sn = *reinterpret_cast<const float4 *>(&cs[1][row][p * kRopePitch + 2 * e]);
                        const float2 c2[2] = {make_float2(co.x, co.y), make_float2(co.z, co.w)};
                        const float2 t2[2] = {make_float2(sn.x, sn.y), make_float2(sn.z, sn.w)};
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float2 minus = make_float2(-t2[i].x, -t2[i].y);
                            const float2 u = f2_fma_rn(x0[e + i], c2[i], f2_mul_rn(x1[e + i], minus));
                            x1[e + i] = f2_fma_rn(x1[e + i], c2[i], f2_mul_rn(x0[e + i], t2[i]));
                            x0[e + i] = u;
                        }
                    }
                }
                const RopeTensor &t = key ? a.k : a.q;
                uint8_t *dst = t.dst + head_offset<VEC>(tok0 + row, t.d_tok, key ? h - a.q.heads : h, t.d_head);
                store8<TYPE, VEC>(dst + e0 * (VEC ? kEs : t.d_dim), t.d_dim, x0);
                store8<TYPE, VEC>(dst + e1 * (VEC ? kEs : t.d_dim), t.d_dim, x1);
            }
        }
        __syncthreads();                           // cos / sin are free for the next tokens
    }
}

template <int TYPE>
void launch(const RopeArgs &a, uint32_t n, bool vec, cudaStream_t st) {
    // a few CTAs an SM, each looping over its rows
    const uint64_t steps = (static_cast<uint64_t>(n) + a.tokens - 1) / a.tokens;
    const uint32_t grid = static_cast<uint32_t>(std::min<uint64_t>(steps, 4ull * num_sms()));
    if (vec) qk_norm_rope_kernel<TYPE, true><<<grid, kRopeThreads, 0, st>>>(a);
    else qk_norm_rope_kernel<TYPE, false><<<grid, kRopeThreads, 0, st>>>(a);
}

bool rope_vec(const kvm_rows *r) { return rows_vec16(r) && ((r->nb_head | r->nb_tok) >> 32) == 0; }

RopeTensor tensor(const kvm_rows *in, const kvm_rows *out, const float *w) {
    RopeTensor t{};
    if (!in) return t;
    t.src = static_cast<const uint8_t *>(in->data);
    t.dst = static_cast<uint8_t *>(const_cast<void *>(out->data));
    t.weight = w;
    t.s_dim = in->nb_dim; t.s_head = in->nb_head; t.s_tok = in->nb_tok;
    t.d_dim = out->nb_dim; t.d_head = out->nb_head; t.d_tok = out->nb_tok;
    t.heads = in->n_head;
    return t;
}

}  // namespace
}  // namespace kvm

using namespace kvm;

extern "C" kvm_status kvm_qk_norm_rope(kvm_stream stream, uint32_t n, const kvm_rows *q, const kvm_rows *k,
                                       const float *d_q_weight, const float *d_k_weight, float eps,
                                       const float *d_freqs, uint32_t n_rot, const int32_t *d_pos,
                                       const kvm_rows *q_out, const kvm_rows *k_out) {
    const char *me = "kvm_qk_norm_rope";
    if (!q || !q_out) return layer_fail(KVM_EINVAL, "%s: null q", me);
    if (!k != !k_out) return layer_fail(KVM_EINVAL, "%s: k and k_out go together", me);
    const uint32_t D = q->head_dim;
    if (D == 0 || D % 16u || D > kRopeMaxDim) return layer_fail(KVM_EINVAL, "%s: head_dim must be a multiple of 16 up to %u", me, kRopeMaxDim);
    if (q->n_head == 0 || q->n_head > 65535u || (k && (k->n_head == 0 || k->n_head > 65535u)))
        return layer_fail(KVM_EINVAL, "%s: 1 to 65535 heads", me);
    if (n_rot % 16u || n_rot > D) return layer_fail(KVM_EINVAL, "%s: n_rot must be a multiple of 16 up to head_dim", me);
    if (n > 0x7fffffffu) return layer_fail(KVM_EINVAL, "%s: too many rows", me);
    if (!(eps >= 0.0f)) return layer_fail(KVM_EINVAL, "%s: eps must not be negative", me);
    if (n_rot && (!d_freqs || !d_pos)) return layer_fail(KVM_EINVAL, "%s: null freqs or pos", me);
    if ((reinterpret_cast<uintptr_t>(d_freqs) | reinterpret_cast<uintptr_t>(d_pos) |
         reinterpret_cast<uintptr_t>(d_q_weight) | reinterpret_cast<uintptr_t>(d_k_weight)) & 3u)
        return layer_fail(KVM_EINVAL, "%s: weights, freqs and pos must be 4-byte aligned", me);
    if (n == 0) return KVM_OK;
    kvm_status r;
    if ((r = rows_check(q, q->n_head, D, "kvm_qk_norm_rope q")) != KVM_OK) return r;
    if ((r = rows_check(q_out, q->n_head, D, "kvm_qk_norm_rope q_out")) != KVM_OK) return r;
    if (k && (r = rows_check(k, k->n_head, D, "kvm_qk_norm_rope k")) != KVM_OK) return r;
    if (k && (r = rows_check(k_out, k->n_head, D, "kvm_qk_norm_rope k_out")) != KVM_OK) return r;
    if (q_out->type != q->type || (k && (k->type != q->type || k_out->type != q->type)))
        return layer_fail(KVM_EINVAL, "%s: q, k and their outputs must have one type", me);
    PointerDevice dev(q->data, me);
    if (dev.status() != KVM_OK) return dev.status();
    RopeArgs a{};
    a.q = tensor(q, q_out, d_q_weight);
    a.k = tensor(k, k_out, d_k_weight);
    a.freqs = d_freqs;
    a.pos = d_pos;
    a.eps = eps;
    a.head_dim = D;
    a.n_rot = n_rot;
    a.lanes = 1;
    while (a.lanes < D / 16u) a.lanes *= 2;
    a.n = n;
    a.inv_dim = 1.0f / static_cast<float>(D);
    // as many rows at a time as keep a thread's batch of heads full, while every SM
    // still has several CTAs' worth
    const uint32_t groups = kRopeThreads / a.lanes, rounds = (a.q.heads + a.k.heads + groups - 1) / groups;
    a.tokens = 1;
    while (a.tokens < kRopeTokens && 2u * a.tokens * rounds <= 4u && n >= 8ull * a.tokens * num_sms()) a.tokens *= 2;
    const bool vec = ((reinterpret_cast<uintptr_t>(d_q_weight) | reinterpret_cast<uintptr_t>(d_k_weight)) & 15u) == 0 && rope_vec(q) && rope_vec(q_out) && (!k || (rope_vec(k) && rope_vec(k_out)));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (q->type == KVM_TYPE_F32) launch<KVM_TYPE_F32>(a, n, vec, st);
    else if (q->type == KVM_TYPE_F16) launch<KVM_TYPE_F16>(a, n, vec, st);
    else launch<KVM_TYPE_BF16>(a, n, vec, st);
    return layer_cuda(cudaGetLastError(), me);
}
