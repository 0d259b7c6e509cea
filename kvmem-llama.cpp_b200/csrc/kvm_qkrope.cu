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
// pair that a rotation mixes (8 values and their partners n_rot/2 further on) of
// several heads of one token: its 8 cos / sin pairs and 16 weights stay in
// registers for all of them, the rotation needs no exchange, and the norm only a
// reduction over the head's head_dim/16 neighbouring threads.  No shared memory
// and no barrier.  A token's heads are split over more threads while the tokens
// alone do not fill the GPU (launch below).
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
    uint32_t n, splits, per_split;     // a token's heads in `splits` ranges of per_split
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

template <bool VEC>
__device__ __forceinline__ void load_weights(const float *w, uint32_t e, float (&x)[8]) {
    if (!w) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 1.0f;
    } else if constexpr (VEC) {
        const float4 a = *reinterpret_cast<const float4 *>(w + e), b = *reinterpret_cast<const float4 *>(w + e + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = w[e + i];
    }
}

template <int TYPE, bool VEC>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
    const uint32_t heads = a.q.heads + a.k.heads;
    const uint64_t unit = (static_cast<uint64_t>(blockIdx.x) * kRopeThreads + threadIdx.x) / a.lanes;   // (token, head range)
    const uint32_t p = threadIdx.x & (a.lanes - 1);
    const uint32_t tok = static_cast<uint32_t>(unit / a.splits), part = static_cast<uint32_t>(unit - static_cast<uint64_t>(tok) * a.splits);
    const uint32_t h0 = part * a.per_split, h1 = min(heads, h0 + a.per_split);
    const bool in = p < a.head_dim / 16 && tok < a.n && h0 < h1;
    const uint32_t half = a.n_rot / 2, pairs = a.n_rot / 16;
    const bool rot = p < pairs;
    // the two chunks of 8 of this thread
    const uint32_t e0 = rot ? 8 * p : a.n_rot + 16 * (p - pairs), e1 = rot ? e0 + half : e0 + 8;
    auto address = [&](uint32_t h, bool out) -> uint64_t {
        const bool key = h >= a.q.heads;
        const RopeTensor &t = key ? a.k : a.q;
        const uint64_t hh = key ? h - a.q.heads : h;
        return out ? reinterpret_cast<uint64_t>(t.dst) + tok * t.d_tok + hh * t.d_head
                   : reinterpret_cast<uint64_t>(t.src) + tok * t.s_tok + hh * t.s_head;
    };
    auto fetch = [&](uint32_t h, float (&x0)[8], float (&x1)[8]) {
        const uint64_t dim = h >= a.q.heads ? a.k.s_dim : a.q.s_dim;
        const uint8_t *src = reinterpret_cast<const uint8_t *>(address(h, false));
        load8<TYPE, VEC>(src + e0 * dim, dim, x0);
        load8<TYPE, VEC>(src + e1 * dim, dim, x1);
    };
    float x0[8], x1[8], n0[8], n1[8], w0[8], w1[8], cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x0[i] = x1[i] = 0.0f;
    if (in) {
        fetch(h0, x0, x1);
        load_weights<VEC>(h0 < a.q.heads ? a.q.weight : a.k.weight, e0, w0);
        load_weights<VEC>(h0 < a.q.heads ? a.q.weight : a.k.weight, e1, w1);
        if (rot) {
            const double pos = static_cast<double>(a.pos[tok]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double ang = pos * static_cast<double>(a.freqs[e0 + i]);
                // in half turns: 1 / pi to 106 bits, its F64 value and the remainder
                const double turn = ang * 0.31830988618379067154;
                const double rest = fma(ang, 0.31830988618379067154, -turn) + ang * -1.9678676675182486e-17;
                const double near = turn - 2.0 * rint(0.5 * turn);
                sincospif(static_cast<float>(near + rest), &sn[i], &cs[i]);
            }
        }
    }
    // every thread of the warp takes the same number of turns (per_split), so the
    // head's threads can reduce with full-warp shuffles
    for (uint32_t j = 0; j < a.per_split; ++j) {
        const uint32_t h = h0 + j;
        const bool on = in && h < h1;
        if (in && h + 1 < h1) fetch(h + 1, n0, n1);
        if (on && h == a.q.heads && j) {
            load_weights<VEC>(a.k.weight, e0, w0);
            load_weights<VEC>(a.k.weight, e1, w1);
        }
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += x0[i] * x0[i] + x1[i] * x1[i];
        for (uint32_t o = a.lanes / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (on) {
            const float rs = rsqrtf(ss / static_cast<float>(a.head_dim) + a.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y0 = x0[i] * rs * w0[i], y1 = x1[i] * rs * w1[i];
                x0[i] = rot ? y0 * cs[i] - y1 * sn[i] : y0;
                x1[i] = rot ? y1 * cs[i] + y0 * sn[i] : y1;
            }
            const uint64_t dim = h >= a.q.heads ? a.k.d_dim : a.q.d_dim;
            uint8_t *dst = reinterpret_cast<uint8_t *>(address(h, true));
            store8<TYPE, VEC>(dst + e0 * dim, dim, x0);
            store8<TYPE, VEC>(dst + e1 * dim, dim, x1);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x0[i] = n0[i];
            x1[i] = n1[i];
        }
    }
}

template <int TYPE>
void launch(const RopeArgs &a, uint32_t n, bool vec, cudaStream_t st) {
    const uint64_t threads = static_cast<uint64_t>(n) * a.splits * a.lanes;
    const uint32_t grid = static_cast<uint32_t>((threads + kRopeThreads - 1) / kRopeThreads);
    if (vec) qk_norm_rope_kernel<TYPE, true><<<grid, kRopeThreads, 0, st>>>(a);
    else qk_norm_rope_kernel<TYPE, false><<<grid, kRopeThreads, 0, st>>>(a);
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
    const uint32_t heads = a.q.heads + a.k.heads;
    const uint64_t fill = 1024ull * num_sms(), have = static_cast<uint64_t>(n) * a.lanes;
    a.n = n;
    a.per_split = heads;
    if (have < fill) a.per_split = static_cast<uint32_t>(std::max<uint64_t>(1, heads * have / fill));
    a.splits = (heads + a.per_split - 1) / a.per_split;
    if (static_cast<uint64_t>(n) * a.splits * a.lanes / kRopeThreads > 0x7ffffff0ull) return layer_fail(KVM_EINVAL, "%s: too many rows", me);
    const bool vec = ((reinterpret_cast<uintptr_t>(d_q_weight) | reinterpret_cast<uintptr_t>(d_k_weight)) & 15u) == 0 && rows_vec16(q) && rows_vec16(q_out) && (!k || (rows_vec16(k) && rows_vec16(k_out)));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (q->type == KVM_TYPE_F32) launch<KVM_TYPE_F32>(a, n, vec, st);
    else if (q->type == KVM_TYPE_F16) launch<KVM_TYPE_F16>(a, n, vec, st);
    else launch<KVM_TYPE_BF16>(a, n, vec, st);
    return layer_cuda(cudaGetLastError(), me);
}
