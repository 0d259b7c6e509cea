// kvm_attend.cu -- kvm_attend: argument checks and the choice of kernel.
#include <algorithm>
#include <cmath>

#include "kvm_attend.cuh"
#include "kvm_layer.cuh"

namespace kvm {

template <int D, int KT>
cudaError_t launch_attend_split(const AttendArgs &a, int vt, int nt, uint32_t grid, cudaStream_t st);
template <int D, int KT>
cudaError_t launch_attend_tile(const AttendArgs &a, int vt, bool pair, uint32_t grid, cudaStream_t st);

bool attend_map(CUtensorMap *map, const void *base, uint64_t row_bytes, const AttendArgs &a, uint32_t box_bytes, uint32_t box_rows) {
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            fn = nullptr;
        }
        return reinterpret_cast<Encode>(fn);
    }();
    if (!encode) return false;
    const cuuint64_t dims[2] = {row_bytes / 4u, static_cast<uint64_t>(a.n_slots) * a.block_tokens};
    const cuuint64_t strides[1] = {row_bytes};
    const cuuint32_t box[2] = {box_bytes / 4u, box_rows}, step[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void *>(base), dims, strides, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

// One of the kernels: split with row tiles of 8 * nt rows, or tile by single CTAs
// (nt = 0) or by pairs (-1).
template <int D, int KT>
cudaError_t launch_kt(const AttendArgs &a, int vt, int nt, uint32_t grid, cudaStream_t st) {
    return nt > 0 ? launch_attend_split<D, KT>(a, vt, nt, grid, st) : launch_attend_tile<D, KT>(a, vt, nt < 0, grid, st);
}

template <int D>
cudaError_t launch_d(const AttendArgs &a, int kt, int vt, int nt, uint32_t grid, cudaStream_t st) {
    switch (kt) {
        case KVM_TYPE_Q4_0: return launch_kt<D, KVM_TYPE_Q4_0>(a, vt, nt, grid, st);
        case KVM_TYPE_Q5_0: return launch_kt<D, KVM_TYPE_Q5_0>(a, vt, nt, grid, st);
        case KVM_TYPE_Q8_0: return launch_kt<D, KVM_TYPE_Q8_0>(a, vt, nt, grid, st);
        default: return launch_kt<D, KVM_TYPE_F16>(a, vt, nt, grid, st);
    }
}

AttendRows rows_of(const kvm_rows *r) {
    return AttendRows{static_cast<const uint8_t *>(r->data), r->nb_dim, r->nb_head, r->nb_tok,
                      r->type == KVM_TYPE_BF16 ? 1 : 0};
}

}  // namespace
}  // namespace kvm

using namespace kvm;

extern "C" kvm_status kvm_attend(kvm_stream stream, const kvm_cache *c, const kvm_attend_batch *b, const kvm_rows *q,
                                 const kvm_rows *out, void *d_work, uint64_t work_bytes) {
    const char *me = "kvm_attend";
    kvm_status r = cache_check(c, me);
    if (r != KVM_OK) return r;
    if (!b || !q || !out) return layer_fail(KVM_EINVAL, "%s: null argument", me);
    const uint32_t D = c->head_dim;
    if (D != 64u && D != 128u && D != 256u) return layer_fail(KVM_EINVAL, "%s: head_dim must be 64, 128 or 256", me);
    if (q->n_head == 0 || q->n_head % c->n_head_kv || q->n_head > 65535u)
        return layer_fail(KVM_EINVAL, "%s: query heads must be a multiple of the %u KV heads", me, c->n_head_kv);
    if (b->n_seq == 0 || b->n_rows == 0) return KVM_OK;
    if ((r = rows_check(q, q->n_head, D, "kvm_attend q")) != KVM_OK) return r;
    if ((r = rows_check(out, q->n_head, D, "kvm_attend out")) != KVM_OK) return r;
    if (q->type == KVM_TYPE_F32 || out->type == KVM_TYPE_F32)
        return layer_fail(KVM_EINVAL, "%s: q and out must be F16 or BF16", me);
    constexpr uint32_t kSkips = KVM_ATTEND_TEST_SKIP_K | KVM_ATTEND_TEST_SKIP_V;
    if (b->flags & ~(KVM_ATTEND_CAUSAL | kSkips)) return layer_fail(KVM_EINVAL, "%s: unknown flags", me);
    if (!std::isfinite(b->scale)) return layer_fail(KVM_EINVAL, "%s: scale must be finite", me);
    if (b->n_seq > 65535u) return layer_fail(KVM_EINVAL, "%s: at most 65535 requests", me);
    if (static_cast<uint64_t>(b->n_rows) * (q->n_head / c->n_head_kv) > 0x7fffffffull || b->table_cols > 0x7fffffffu)
        return layer_fail(KVM_EINVAL, "%s: too many rows or columns", me);
    if (b->n_seq > 1 && b->table_stride < b->table_cols) return layer_fail(KVM_EINVAL, "%s: table_stride < table_cols", me);
    if (b->n_seq && (!b->d_q_start || !b->d_kv_len || (b->table_cols && !b->d_table)))
        return layer_fail(KVM_EINVAL, "%s: null buffer", me);
    if ((reinterpret_cast<uintptr_t>(b->d_table) | reinterpret_cast<uintptr_t>(b->d_q_start) |
         reinterpret_cast<uintptr_t>(b->d_kv_len)) & 3u)
        return layer_fail(KVM_EINVAL, "%s: table, q_start and kv_len must be 4-byte aligned", me);
    if (!d_work || work_bytes < KVM_ATTEND_WORK_BYTES || (reinterpret_cast<uintptr_t>(d_work) & 15u))
        return layer_fail(KVM_EINVAL, "%s: workspace must be %u bytes, 16-byte aligned", me, KVM_ATTEND_WORK_BYTES);
    PointerDevice dev(c->d_k, me);
    if (dev.status() != KVM_OK) return dev.status();

    AttendArgs a{};
    const uint32_t width = c->n_head_kv * D;
    a.k = static_cast<const uint8_t *>(c->d_k);
    a.v = static_cast<const uint8_t *>(c->d_v);
    a.row_k = kvm_row_bytes(c->type_k, width);
    a.row_v = kvm_row_bytes(c->type_v, width);
    a.table = b->d_table;
    a.table_stride = b->table_stride;
    a.table_cols = b->table_cols;
    a.q_start = b->d_q_start;
    a.kv_len = b->d_kv_len;
    a.n_seq = b->n_seq;
    a.n_rows = b->n_rows;
    a.n_head_kv = c->n_head_kv;
    a.group = q->n_head / c->n_head_kv;
    a.block_tokens = c->block_tokens;
    a.n_slots = c->n_slots;
    a.block_shift = 32;
    for (uint32_t s = 0; s < 32; ++s)
        if (c->block_tokens == 1u << s) a.block_shift = s;
    a.scale_log2 = b->scale * 1.4426950408889634f;
    a.causal = (b->flags & KVM_ATTEND_CAUSAL) ? 1u : 0u;
    a.skip = b->flags & kSkips;
    a.q = rows_of(q);
    a.out = rows_of(out);
    a.work = static_cast<uint8_t *>(d_work);
    a.align16 = ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | a.row_k | a.row_v) & 15u) == 0;
    a.tma = a.align16 && c->block_tokens % kAttendBox == 0;
    a.q_vec = rows_vec16(q);
    a.out_vec = rows_vec16(out);
    a.max_keys = static_cast<uint32_t>(std::min<uint64_t>(static_cast<uint64_t>(b->table_cols) * c->block_tokens, 0x7fffffffu));
    a.heads_cta = c->n_head_kv % 4u == 0 ? 4 : c->n_head_kv % 2u == 0 ? 2 : 1;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const uint64_t sms = static_cast<uint64_t>(num_sms());
    // no more CTAs than the call can have work for: row tiles of r rows, steps of k keys
    auto ctas = [&](uint32_t r, uint32_t k, uint32_t heads) -> uint32_t {
        const uint64_t tiles = static_cast<uint64_t>(b->n_rows) * a.group / r + b->n_seq;
        const uint64_t steps = (static_cast<uint64_t>(b->table_cols) * c->block_tokens + k - 1) / k + 1;
        const uint64_t items = tiles * (c->n_head_kv / heads);
        uint64_t n = std::min<uint64_t>(sms, kAttendMaxCtas);
        if (items < n && steps < n) n = std::min(n, items * steps);
        return static_cast<uint32_t>(std::max<uint64_t>(n, 1));
    };
    auto launch = [&](int nt, uint32_t min_rows, uint32_t max_rows) {
        a.min_rows = min_rows;
        a.max_rows = max_rows;
        const uint32_t grid = nt > 0 ? ctas(8u * nt, 16u, a.heads_cta) : nt == 0 ? ctas(128, 64, 1) :
                                                                                 static_cast<uint32_t>(std::min<uint64_t>(2u * ctas(256, 128, 1), sms & ~1ull));
        if (D == 64u) return launch_d<64>(a, c->type_k, c->type_v, nt, grid, st);
        if (D == 128u) return launch_d<128>(a, c->type_k, c->type_v, nt, grid, st);
        return launch_d<256>(a, c->type_k, c->type_v, nt, grid, st);
    };
    // Requests of up to 16 query rows go to the split kernel, longer ones to the tile
    // kernel; the device sorts them, so a wrong max_new costs time and the tile kernel's
    // roundings, nothing else.  Alike requests (one, or drafts that fit a row tile with more
    // than 8 rows on average) take one kernel, since the tile kernel's time hardly depends
    // on the rows in a tile: 24 rows of 32 alike requests of 2048 keys 89 us, in row tiles of
    // 8 112, of 16 135.
    // Few requests do better in row tiles of 8 (24 query and 4 KV heads of 256, us; the borders
    // were set on this layer): 12 rows of 1 request of 32768 keys 34, in tiles of 16 39; 8 of
    // 16385 94 and 103; 32 of 1024 42 and 33.  24 rows of 1 request of 32768 keys 42, in the tile
    // kernel 60; 2 of up to 8192 30 and 43; 4 alike of 2048 31 and 27, 8 alike of 16384 138 and
    // 134, but 8 of all lengths up to that 76 and 87.  8 KV heads of 128, q8_0, 24 rows of 8
    // alike requests of 2048: 49 and 40.
    const uint64_t most = static_cast<uint64_t>(b->max_new) * a.group;
    cudaError_t e;
    if (most <= 16u || (most <= 24u && b->n_seq <= 3u)) {
        e = launch(most <= 8u || b->n_seq <= 8u ? 1 : 2, 1, 0xffffffffu);
    } else if (b->n_seq == 1 || (most <= 128u && static_cast<uint64_t>(b->n_rows) * a.group > 8ull * b->n_seq)) {
        e = launch(most > 128u ? -1 : 0, 1, 0xffffffffu);
    } else {
        e = launch(2, 1, 16);
        if (e == cudaSuccess) e = launch(most > 128u ? -1 : 0, 17, 0xffffffffu);
    }
    return layer_cuda(e, me);
}
