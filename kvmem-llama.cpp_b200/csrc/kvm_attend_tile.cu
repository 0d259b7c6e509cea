// kvm_attend_tile.cu -- the instances of attend_tile_kernel for one head size and
// K type (compiled once for each pair of KVM_ATTEND_D, KVM_ATTEND_KT).
#include <algorithm>

#include "kvm_attend_tile.cuh"

namespace kvm {
namespace {

template <int D, int KT, int VT, bool PAIR>
cudaError_t launch(AttendArgs a, uint32_t grid, cudaStream_t st) {
    using G = TileGeom<D, KT, VT, PAIR>;
    static std::atomic<uint64_t> attr{0};
    static_assert(G::kSmem <= 222 * 1024, "shared memory");       // beside it the kernel's static 5 KB
    const auto kernel = [] {
        if constexpr (PAIR) return attend_pair_kernel<D, KT, VT>;
        else return attend_tile_kernel<D, KT, VT>;
    }();
    if (!attr_once(attr, reinterpret_cast<const void *>(kernel), G::kSmem)) return cudaErrorInvalidValue;
    if (a.tma && !(attend_map(&a.map_k, a.k, a.row_k, a, G::K::kStride, kAttendBox) && attend_map(&a.map_v, a.v, a.row_v, a, G::V::kStride, kAttendBox)))
        a.tma = 0;
    // units: CTAs, or pairs of them
    constexpr uint32_t kCtas = PAIR ? 2 : 1;
    const uint32_t units = std::max(1u, std::min<uint32_t>(grid / kCtas, (KVM_ATTEND_WORK_BYTES - kAttendMaxCtas * kAttendDescBytes) /
                                                                            (2u * tile_part_bytes<D, G::kRows>())));
    kernel<<<units * kCtas, kTileThreads, G::kSmem, st>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || units == 1) return e;
    return launch_after_prev(attend_tile_join_kernel<D, G::kRows>, dim3(std::min<uint32_t>(2u * num_sms(), units * G::kRows)),
                             dim3(kJoinThreads), 0, st, a, units);
}

// Pairs where they exist (see TileGeom: quantized K and V of 128 or 256 dims whose
// rows fit beside the operands) and the requests are long enough.
template <int D, int KT, int VT>
cudaError_t launch_any(const AttendArgs &a, bool pair, uint32_t grid, cudaStream_t st) {
    if constexpr (D >= 128 && KT != KVM_TYPE_F16 && VT != KVM_TYPE_F16) {
        using G = TileGeom<D, KT, VT, true>;
        if constexpr (G::kFit >= 1)
            if (pair && grid >= 2) return launch<D, KT, VT, true>(a, grid, st);
    }
    return launch<D, KT, VT, false>(a, grid, st);
}

}  // namespace

template <int D, int KT>
cudaError_t launch_attend_tile(const AttendArgs &a, int vt, bool pair, uint32_t grid, cudaStream_t st) {
    switch (vt) {
        case KVM_TYPE_Q4_0: return launch_any<D, KT, KVM_TYPE_Q4_0>(a, pair, grid, st);
        case KVM_TYPE_Q5_0: return launch_any<D, KT, KVM_TYPE_Q5_0>(a, pair, grid, st);
        case KVM_TYPE_Q8_0: return launch_any<D, KT, KVM_TYPE_Q8_0>(a, pair, grid, st);
        default: return launch_any<D, KT, KVM_TYPE_F16>(a, pair, grid, st);
    }
}
template cudaError_t launch_attend_tile<KVM_ATTEND_D, KVM_ATTEND_KT>(const AttendArgs &, int, bool, uint32_t, cudaStream_t);

}  // namespace kvm
