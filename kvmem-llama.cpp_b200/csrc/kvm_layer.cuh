// kvm_layer.cuh -- host helpers shared by the sessionless calls of the
// attention layer (kvm_map_batch, kvm_qk_norm_rope, kvm_write_rows,
// kvm_read_rows, kvm_attend).
#pragma once

#include <cstdarg>
#include <cstdio>

#include "kvm_internal.cuh"
#include "kvm_quant.cuh"

namespace kvm {

void set_sessionless_error(const char *msg);

inline kvm_status layer_fail(kvm_status st, const char *fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    set_sessionless_error(buf);
    return st;
}

inline kvm_status layer_cuda(cudaError_t e, const char *what) {
    if (e == cudaSuccess) return KVM_OK;
    return layer_fail(e == cudaErrorMemoryAllocation ? KVM_ENOMEM : KVM_ECUDA, "%s: %s", what,
                      cudaGetErrorString(e));
}

// Makes the device of a pointer current for the call.
class PointerDevice {
public:
    explicit PointerDevice(const void *p, const char *what) {
        cudaPointerAttributes at{};
        const cudaError_t e = cudaPointerGetAttributes(&at, p);
        if (e != cudaSuccess) {
            cudaGetLastError();
            st_ = layer_fail(KVM_ECUDA, "%s: %s", what, cudaGetErrorString(e));
            return;
        }
        if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) {
            st_ = layer_fail(KVM_EINVAL, "%s: not a device pointer", what);
            return;
        }
        int cur = -1;
        if (cudaGetDevice(&cur) == cudaSuccess && cur != at.device) {
            if (cudaSetDevice(at.device) != cudaSuccess) {
                cudaGetLastError();
                st_ = layer_fail(KVM_ECUDA, "%s: cannot use device %d", what, at.device);
                return;
            }
            prev_ = cur;
        }
    }
    ~PointerDevice() {
        if (prev_ >= 0) cudaSetDevice(prev_);
    }
    PointerDevice(const PointerDevice &) = delete;
    PointerDevice &operator=(const PointerDevice &) = delete;
    kvm_status status() const { return st_; }

private:
    int prev_ = -1;
    kvm_status st_ = KVM_OK;
};

inline bool act_type_ok(int32_t t) { return t == KVM_TYPE_F32 || t == KVM_TYPE_F16 || t == KVM_TYPE_BF16; }
inline uint32_t act_bytes(int32_t t) { return t == KVM_TYPE_F32 ? 4u : 2u; }
inline bool cache_type_ok(int32_t t) {
    return t == KVM_TYPE_F16 || t == KVM_TYPE_Q8_0 || t == KVM_TYPE_Q4_0 || t == KVM_TYPE_Q5_0;
}

// One activation tensor: type, shape, and strides that keep every element
// aligned to its size.
inline kvm_status rows_check(const kvm_rows *r, uint32_t n_head, uint32_t head_dim, const char *what) {
    if (!r || !r->data) return layer_fail(KVM_EINVAL, "%s: null tensor", what);
    if (!act_type_ok(r->type)) return layer_fail(KVM_EINVAL, "%s: type must be F32, F16 or BF16", what);
    if (r->n_head != n_head || r->head_dim != head_dim)
        return layer_fail(KVM_EINVAL, "%s: %u heads of %u, expected %u of %u", what, r->n_head, r->head_dim, n_head,
                          head_dim);
    const uint64_t es = act_bytes(r->type);
    if ((reinterpret_cast<uintptr_t>(r->data) | r->nb_dim | r->nb_head | r->nb_tok) & (es - 1))
        return layer_fail(KVM_EINVAL, "%s: data and strides must be multiples of the element size", what);
    return KVM_OK;
}

// 16-byte vectors along the head: contiguous values, everything aligned.
inline bool rows_vec16(const kvm_rows *r) {
    return r->nb_dim == act_bytes(r->type) &&
           ((reinterpret_cast<uintptr_t>(r->data) | r->nb_head | r->nb_tok) & 15u) == 0;
}

inline kvm_status cache_check(const kvm_cache *c, const char *what) {
    if (!c || !c->d_k || !c->d_v) return layer_fail(KVM_EINVAL, "%s: null cache", what);
    if (!cache_type_ok(c->type_k) || !cache_type_ok(c->type_v))
        return layer_fail(KVM_EINVAL, "%s: cache types must be F16, Q8_0, Q5_0 or Q4_0", what);
    if (c->n_head_kv == 0 || c->n_head_kv > kMaxHeadsKv || c->head_dim == 0 || c->head_dim % 32u || c->head_dim > kMaxHeadDim)
        return layer_fail(KVM_EINVAL, "%s: 1 to %u KV heads of a multiple of 32 up to %u", what, kMaxHeadsKv, kMaxHeadDim);
    if (c->block_tokens == 0 || c->n_slots == 0 ||
        static_cast<uint64_t>(c->block_tokens) * c->n_slots > 0x7fffffffull)
        return layer_fail(KVM_EINVAL, "%s: block_tokens * n_slots must be 1 to 2^31 - 1", what);
    if ((reinterpret_cast<uintptr_t>(c->d_k) | reinterpret_cast<uintptr_t>(c->d_v)) & 3u)
        return layer_fail(KVM_EINVAL, "%s: cache bases must be 4-byte aligned", what);
    return KVM_OK;
}

}  // namespace kvm
