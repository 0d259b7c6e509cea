// kvm_qkrope.cu -- kvm_qk_norm_rope: RMS norm of every query and key head and
// the NeoX rotation, one pass over the values.
//
//   y = x * rsqrt(mean(x^2) + eps) * w;   (y_i, y_{i+h}) -> (y_i c - y_{i+h} s, y_{i+h} c + y_i s)
//
// h = n_rot / 2, (c, s) = cos, sin of pos * freq_i.  The angle is a product of
// an integer and an F32 value, exact in F64 up to 2^29 and within 2^-53 beyond;
// it is reduced by multiples of 2 pi in F64 (a far position would lose every
// digit in F32) and only the remainder goes to F32.  Norm, rotation and sums
// are F32 and each value is rounded once, at the store.
//
// Bound by HBM: every value is read and written once.  One CTA a token: its
// cos / sin are formed once in shared memory for all heads, while the CTA's
// first loads are in flight.  A thread owns the chunk pair that a rotation mixes (8
// values and their partners n_rot/2 further on), so the rotation needs no
// exchange and the norm only a reduction over the head's head_dim/16 threads.
#include <cuda_bf16.h>

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
};

template <int TYPE, bool VEC>
__device__ __forceinline__ void load8(const uint8_t *p, uint64_t nb_dim, float (&x)[8]) {
    if constexpr (VEC && TYPE == KVM_TYPE_F32) {
        const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 16);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else if constexpr (VEC) {
        const uint4 r = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (TYPE == KVM_TYPE_F16) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            } else {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint8_t *e = p + i * nb_dim;
            if constexpr (TYPE == KVM_TYPE_F32) x[i] = *reinterpret_cast<const float *>(e);
            else if constexpr (TYPE == KVM_TYPE_F16) x[i] = __half2float(*reinterpret_cast<const __half *>(e));
            else x[i] = __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(e)) << 16);
        }
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
__device__ __forceinline__ void store8(uint8_t *p, uint64_t nb_dim, const float (&x)[8]) {
    if constexpr (VEC && TYPE == KVM_TYPE_F32) {
        *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4 *>(p + 16) = make_float4(x[4], x[5], x[6], x[7]);
    } else if constexpr (VEC) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack2<TYPE>(x[0], x[1]), pack2<TYPE>(x[2], x[3]),
                                                   pack2<TYPE>(x[4], x[5]), pack2<TYPE>(x[6], x[7]));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint8_t *e = p + i * nb_dim;
            if constexpr (TYPE == KVM_TYPE_F32) *reinterpret_cast<float *>(e) = x[i];
            else *reinterpret_cast<uint16_t *>(e) = static_cast<uint16_t>(pack2<TYPE>(x[i], 0.0f) & 0xffffu);
        }
    }
}

template <int TYPE, bool VEC>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
    __shared__ float2 turn[kRopeMaxDim / 2];
    const uint32_t tok = blockIdx.x;
    const uint32_t half = a.n_rot / 2, pairs = a.n_rot / 16;
    const uint32_t p = threadIdx.x & (a.lanes - 1), per_pass = kRopeThreads / a.lanes;
    const uint32_t heads = a.q.heads + a.k.heads;
    const bool in = p < a.head_dim / 16;
    const bool rot = p < pairs;
    // the two chunks of 8 of this thread
    const uint32_t e0 = rot ? 8 * p : a.n_rot + 16 * (p - pairs), e1 = rot ? e0 + half : e0 + 8;
    uint32_t h = threadIdx.x / a.lanes;
    float x0[8], x1[8];
    auto fetch = [&](uint32_t hh) {
        const bool key = hh >= a.q.heads;
        const RopeTensor &t = key ? a.k : a.q;
        const uint8_t *src = t.src + tok * t.s_tok + static_cast<uint64_t>(key ? hh - a.q.heads : hh) * t.s_head;
        load8<TYPE, VEC>(src + e0 * t.s_dim, t.s_dim, x0);
        load8<TYPE, VEC>(src + e1 * t.s_dim, t.s_dim, x1);
    };
    if (in && h < heads) fetch(h);
    if (half) {
        const double pos = static_cast<double>(a.pos[tok]);
        for (uint32_t i = threadIdx.x; i < half; i += kRopeThreads) {
            const double ang = pos * static_cast<double>(a.freqs[i]);
            // 2 pi to 106 bits: its F64 value and the remainder
            const double k = rint(ang * 0.15915494309189533577);
            const double r = fma(-k, 2.4492935982947064e-16, fma(-k, 6.2831853071795864769, ang));
            float sn, cs;
            sincosf(static_cast<float>(r), &sn, &cs);
            turn[i] = make_float2(cs, sn);
        }
        __syncthreads();
    }
    for (; h < heads; h += per_pass) {
        const bool key = h >= a.q.heads;
        const RopeTensor &t = key ? a.k : a.q;
        float ss = 0.0f;
        if (in) {
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += x0[i] * x0[i] + x1[i] * x1[i];
        }
        // the threads of a head are neighbours in a warp and leave the loop together
        for (uint32_t o = a.lanes / 2; o; o >>= 1) ss += __shfl_xor_sync(__activemask(), ss, o);
        const float rs = rsqrtf(ss / static_cast<float>(a.head_dim) + a.eps);
        if (in) {
            float y0[8], y1[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y0[i] = x0[i] * rs * (t.weight ? t.weight[e0 + i] : 1.0f);
                y1[i] = x1[i] * rs * (t.weight ? t.weight[e1 + i] : 1.0f);
            }
            if (rot) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 cs = turn[e0 + i];
                    const float u = y0[i] * cs.x - y1[i] * cs.y;
                    y1[i] = y1[i] * cs.x + y0[i] * cs.y;
                    y0[i] = u;
                }
            }
            uint8_t *dst = t.dst + tok * t.d_tok + static_cast<uint64_t>(key ? h - a.q.heads : h) * t.d_head;
            if (h + per_pass < heads) fetch(h + per_pass);
            store8<TYPE, VEC>(dst + e0 * t.d_dim, t.d_dim, y0);
            store8<TYPE, VEC>(dst + e1 * t.d_dim, t.d_dim, y1);
        }
    }
}

template <int TYPE>
void launch(const RopeArgs &a, uint32_t n, bool vec, cudaStream_t st) {
    if (vec) qk_norm_rope_kernel<TYPE, true><<<n, kRopeThreads, 0, st>>>(a);
    else qk_norm_rope_kernel<TYPE, false><<<n, kRopeThreads, 0, st>>>(a);
}

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
    const bool vec = rows_vec16(q) && rows_vec16(q_out) && (!k || (rows_vec16(k) && rows_vec16(k_out)));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (q->type == KVM_TYPE_F32) launch<KVM_TYPE_F32>(a, n, vec, st);
    else if (q->type == KVM_TYPE_F16) launch<KVM_TYPE_F16>(a, n, vec, st);
    else launch<KVM_TYPE_BF16>(a, n, vec, st);
    return layer_cuda(cudaGetLastError(), me);
}
