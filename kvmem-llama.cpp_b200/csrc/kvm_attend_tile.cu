// kvm_attend_tile.cu -- the instances of attend_tile_kernel for one head size and
// K type (compiled once for each pair of KVM_ATTEND_D, KVM_ATTEND_KT).
#include <algorithm>

#include "kvm_attend_tile.cuh"

namespace kvm {
namespace {

template <int D, int KT, int VT>
cudaError_t launch(AttendArgs a, uint32_t grid, cudaStream_t st) {
    using G = TileGeom<D, KT, VT>;
    static std::atomic<uint64_t> attr{0};
    static_assert(G::kSmem <= 227 * 1024, "shared memory");
    if (!attr_once(attr, reinterpret_cast<const void *>(attend_tile_kernel<D, KT, VT>), G::kSmem)) return cudaErrorInvalidValue;
    if (a.tma && !(attend_map(&a.map_k, a.k, a.row_k, a, G::K::kStride, kAttendBox) && attend_map(&a.map_v, a.v, a.row_v, a, G::V::kStride, kAttendBox)))
        a.tma = 0;
    grid = std::min<uint32_t>(grid, (KVM_ATTEND_WORK_BYTES - kAttendMaxCtas * kAttendDescBytes) / (2u * tile_part_bytes<D>()));
    attend_tile_kernel<D, KT, VT><<<grid, kTileThreads, G::kSmem, st>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || grid == 1) return e;
    return launch_after_prev(attend_tile_join_kernel<D>, dim3(std::min<uint32_t>(2u * num_sms(), grid * kTileRows)), dim3(kJoinThreads), 0, st, a, grid);
}

}  // namespace

template <int D, int KT>
cudaError_t launch_attend_tile(const AttendArgs &a, int vt, uint32_t grid, cudaStream_t st) {
    switch (vt) {
        case KVM_TYPE_Q4_0: return launch<D, KT, KVM_TYPE_Q4_0>(a, grid, st);
        case KVM_TYPE_Q5_0: return launch<D, KT, KVM_TYPE_Q5_0>(a, grid, st);
        case KVM_TYPE_Q8_0: return launch<D, KT, KVM_TYPE_Q8_0>(a, grid, st);
        default: return launch<D, KT, KVM_TYPE_F16>(a, grid, st);
    }
}
template cudaError_t launch_attend_tile<KVM_ATTEND_D, KVM_ATTEND_KT>(const AttendArgs &, int, uint32_t, cudaStream_t);

}  // namespace kvm
