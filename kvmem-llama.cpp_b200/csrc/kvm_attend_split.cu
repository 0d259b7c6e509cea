// kvm_attend_split.cu -- the instances of attend_split_kernel for one head size
// and K type (compiled once for each pair of KVM_ATTEND_D, KVM_ATTEND_KT).
#include <algorithm>

#include "kvm_attend_split.cuh"

namespace kvm {

namespace {

template <int D, int KT, int VT, int NT>
cudaError_t launch(AttendArgs a, uint32_t grid, cudaStream_t st) {
    static std::atomic<uint64_t> attr{0};
    using G = SplitGeom<D, KT, VT, NT>;
    constexpr int smem = G::kSmem;
    static_assert(smem <= 227 * 1024, "shared memory");
    if (!attr_once(attr, reinterpret_cast<const void *>(attend_split_kernel<D, KT, VT, NT>), smem))
        return cudaErrorInvalidValue;
    if (a.tma && !(attend_map(&a.map_k, a.k, a.row_k, a, G::K::kStride, kAttendBox) && attend_map(&a.map_v, a.v, a.row_v, a, G::V::kStride, kAttendBox)))
        a.tma = 0;
    // Windows of a few steps a warp (kAttendWholeSteps) whose (request, head) pairs are
    // hardly more than the SMs: a KV head a CTA, nothing cut.  A CTA then begins one or two
    // segments instead of parts of several, and there is no join: 2 requests of 333 keys
    // (4 heads of 256) 27 us by four heads a CTA, cut, and 13.6 us so; 64 of 1024 55 and
    // 39 us; 2 of 1024 22.6 and 20.4.
    const uint64_t steps = (a.max_keys + static_cast<uint64_t>(G::kStep) - 1u) / G::kStep;
    const bool alone = steps <= static_cast<uint64_t>(kAttendWholeSteps * G::kWarps) && static_cast<uint64_t>(a.n_seq) * a.n_head_kv <= 2u * num_sms();
    if (alone) {
        a.heads_cta = 1;
        grid = std::min<uint32_t>(num_sms(), kAttendMaxCtas);
    }
    const uint64_t slot = static_cast<uint64_t>(a.heads_cta) * attend_part_floats<D, NT>() * 4u;
    grid = static_cast<uint32_t>(std::min<uint64_t>(grid, (KVM_ATTEND_WORK_BYTES - kAttendMaxCtas * kAttendDescBytes) / (2 * slot)));
    // segments that the least share would hold whole are not cut at all
    a.whole = alone || steps <= static_cast<uint64_t>(kAttendMinSteps / G::kTiles * (G::kWarps / a.heads_cta));
    attend_split_kernel<D, KT, VT, NT><<<grid, G::kThreads, smem, st>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || grid == 1 || a.whole) return e;
    return launch_after_prev(attend_join_kernel<D, NT>, dim3(std::min<uint32_t>(2u * num_sms(), grid * 8u * NT * a.heads_cta * (D / 64))), dim3(kJoinThreads), 0, st, a, grid);
}

template <int D, int KT, int VT>
cudaError_t launch_nt(const AttendArgs &a, int nt, uint32_t grid, cudaStream_t st) {
    return nt == 1 ? launch<D, KT, VT, 1>(a, grid, st) : launch<D, KT, VT, 2>(a, grid, st);
}

}  // namespace

template <int D, int KT>
cudaError_t launch_attend_split(const AttendArgs &a, int vt, int nt, uint32_t grid, cudaStream_t st) {
    switch (vt) {
        case KVM_TYPE_Q4_0: return launch_nt<D, KT, KVM_TYPE_Q4_0>(a, nt, grid, st);
        case KVM_TYPE_Q5_0: return launch_nt<D, KT, KVM_TYPE_Q5_0>(a, nt, grid, st);
        case KVM_TYPE_Q8_0: return launch_nt<D, KT, KVM_TYPE_Q8_0>(a, nt, grid, st);
        default: return launch_nt<D, KT, KVM_TYPE_F16>(a, nt, grid, st);
    }
}
template cudaError_t launch_attend_split<KVM_ATTEND_D, KVM_ATTEND_KT>(const AttendArgs &, int, int, uint32_t,
                                                                      cudaStream_t);

}  // namespace kvm
