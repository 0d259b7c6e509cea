// kvm_batch.cu -- kvm_map_batch: block tables and the cell map of a step from
// the requests' lengths.
//
// With held = ceil(past/T) and need = ceil((past+new)/T) - held, the inclusive
// sums of need place every request in the free list and those of new give its
// rows, so nothing is sequential: a request runs when it needs no slot or its
// sum fits.  One launch: every CTA repeats the two scans over the (at most
// 4096) requests in shared memory, then the CTAs share the rows -- each row
// finds its request by bisection of the row starts -- and, a warp a request, the
// table entries.  A row's slot comes from the free list itself when its block
// is new, so no CTA waits for another's table writes.
//
// Bound by latency at every size met: a decode step of 64 requests is one CTA's
// two dependent loads, two scans and one store.
// 64 requests: 4.8 us; 512 ragged prompts of up to 1024 tokens (263,000 rows): 9.7 us
// for 4.2 MB.  Sums a warp at a time before the shared atomics: 64-bit atomics of
// every thread took it to 18.5.
#include <algorithm>

#include "kvm_layer.cuh"

namespace kvm {
namespace {

constexpr int kMapThreads = 512;
constexpr uint32_t kMapMaxSeq = 4096;

struct MapSmem {
    int32_t start[kMapMaxSeq + 1];   // first row
    int32_t first[kMapMaxSeq];       // place of the first new slot in the free list, -1 = does not run
};

// Inclusive scan of one 64-bit value a thread; *total gets the sum.
__device__ __forceinline__ uint64_t scan64(uint64_t v, uint64_t *warp_sums, uint64_t *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kMapThreads / 32; ++w) {
        if (w < warp) before += warp_sums[w];
        all += warp_sums[w];
    }
    *total = all;
    __syncthreads();
    return v + before;
}

__global__ void __launch_bounds__(kMapThreads) map_batch_kernel(const __grid_constant__ kvm_batch_map m) {
    __shared__ MapSmem s;
    __shared__ uint64_t sums[kMapThreads / 32];
    __shared__ uint32_t s_idle, s_tokens, s_taken;
    const int tid = threadIdx.x;
    const uint32_t T = m.block_tokens;
    const bool lead = blockIdx.x == 0;
    if (tid == 0) {
        s_idle = s_tokens = s_taken = 0;
        s.start[0] = 0;
    }
    __syncthreads();
    uint64_t row_carry = 0, need_carry = 0;
    for (uint32_t base = 0; base < m.n_seq; base += kMapThreads) {
        const uint32_t i = base + tid;
        const bool in = i < m.n_seq;
        const int64_t past = in ? m.d_past[i] : 0, fresh = in ? m.d_new[i] : 0;
        const uint64_t rows = fresh > 0 ? fresh : 0;
        uint64_t all;
        const uint64_t end = row_carry + scan64(rows, sums, &all);
        row_carry += all;
        const uint64_t held = past > 0 ? (past + T - 1) / T : 0;
        const uint64_t blocks = past >= 0 && fresh >= 0 ? (past + fresh + T - 1) / T : 0;
        const bool good = past >= 0 && fresh >= 0 && blocks <= m.table_cols && (rows == 0 || end <= m.n_rows) &&
                          past + fresh <= 0x7fffffffll;
        const uint64_t need = in && good ? blocks - held : 0;
        const uint64_t upto = need_carry + scan64(need, sums, &all);
        need_carry += all;
        const bool runs = in && good && (need == 0 || upto <= m.n_free);
        if (in) {
            s.start[i + 1] = static_cast<int32_t>(min(end, static_cast<uint64_t>(m.n_rows)));
            // a request that needs nothing may stand past the free list: any place will do
            s.first[i] = !runs ? -1 : need ? static_cast<int32_t>(upto - need) : 0;
            if (lead) {
                m.d_q_start[i + 1] = s.start[i + 1];
                m.d_kv_len[i] = runs ? static_cast<int32_t>(past + fresh) : 0;
            }
        }
        if (lead) {           // sums of a warp first: one shared atomic a warp
            const uint32_t idle = __popc(__ballot_sync(0xffffffffu, in && !runs));
            const uint32_t tokens = __reduce_add_sync(0xffffffffu, runs ? static_cast<uint32_t>(fresh) : 0u);
            const uint32_t taken = __reduce_add_sync(0xffffffffu, runs ? static_cast<uint32_t>(need) : 0u);
            if ((tid & 31) == 0) {
                atomicAdd(&s_idle, idle);
                atomicAdd(&s_tokens, tokens);
                atomicAdd(&s_taken, taken);
            }
        }
    }
    __syncthreads();
    if (lead && tid == 0) {
        m.d_q_start[0] = 0;
        m.d_info[0] = static_cast<int32_t>(s_taken);
        m.d_info[1] = s.start[m.n_seq];
        m.d_info[2] = static_cast<int32_t>(s_idle);
        m.d_info[3] = static_cast<int32_t>(s_tokens);
    }
    // table entries of new blocks, a warp a request
    const uint32_t warps = gridDim.x * (kMapThreads / 32);
    for (uint32_t i = blockIdx.x * (kMapThreads / 32) + (tid >> 5); i < m.n_seq; i += warps) {
        const int32_t first = s.first[i];
        if (first < 0) continue;
        const uint32_t past = m.d_past[i], upto = past + static_cast<uint32_t>(m.d_new[i]);
        const uint32_t held = past / T + (past % T != 0), blocks = upto / T + (upto % T != 0);
        for (uint32_t b = held + (tid & 31); b < blocks; b += 32)
            m.d_table[i * m.table_stride + b] = m.d_free[first + (b - held)];
    }
    // the rows
    const uint32_t rows = static_cast<uint32_t>(s.start[m.n_seq]);
    for (uint32_t r = blockIdx.x * kMapThreads + tid; r < m.n_rows; r += gridDim.x * kMapThreads) {
        int64_t cell = -1;
        int32_t pos = 0, seq = -1;
        if (r < rows) {
            uint32_t lo = 0, hi = m.n_seq;       // the last request with start <= r
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (static_cast<uint32_t>(s.start[mid]) <= r) lo = mid;
                else hi = mid;
            }
            seq = static_cast<int32_t>(lo);
            const uint32_t past = static_cast<uint32_t>(m.d_past[lo]);
            const uint32_t p = past + (r - static_cast<uint32_t>(s.start[lo]));
            pos = static_cast<int32_t>(p);
            const int32_t first = s.first[lo];
            if (first >= 0) {
                const uint32_t b = p / T, held = past / T + (past % T != 0);
                const int32_t slot = b < held ? m.d_table[lo * m.table_stride + b] : m.d_free[first + (b - held)];
                if (slot >= 0) cell = static_cast<int64_t>(slot) * T + (p - b * T);
            }
        }
        m.d_cells[r] = cell;
        m.d_pos[r] = pos;
        m.d_seq[r] = seq;
    }
}

}  // namespace
}  // namespace kvm

using namespace kvm;

extern "C" kvm_status kvm_map_batch(kvm_stream stream, const kvm_batch_map *m) {
    const char *me = "kvm_map_batch";
    if (!m) return layer_fail(KVM_EINVAL, "%s: null argument", me);
    if (m->n_seq == 0 || m->n_seq > kMapMaxSeq) return layer_fail(KVM_EINVAL, "%s: 1 to %u requests", me, kMapMaxSeq);
    if (m->block_tokens == 0 || m->block_tokens > 0x40000000u) return layer_fail(KVM_EINVAL, "%s: bad block_tokens", me);
    if (m->n_rows > 0x7fffffffu || m->n_free > 0x7fffffffu || m->table_cols > 0x7fffffffu)
        return layer_fail(KVM_EINVAL, "%s: n_rows, n_free and table_cols must be below 2^31", me);
    if (m->table_stride < m->table_cols) return layer_fail(KVM_EINVAL, "%s: table_stride < table_cols", me);
    if (!m->d_past || !m->d_new || !m->d_q_start || !m->d_kv_len || !m->d_info || (m->n_free && !m->d_free) ||
        (m->table_cols && !m->d_table) || (m->n_rows && (!m->d_cells || !m->d_pos || !m->d_seq)))
        return layer_fail(KVM_EINVAL, "%s: null buffer", me);
    const uintptr_t low = reinterpret_cast<uintptr_t>(m->d_past) | reinterpret_cast<uintptr_t>(m->d_new) |
                          reinterpret_cast<uintptr_t>(m->d_free) | reinterpret_cast<uintptr_t>(m->d_table) |
                          reinterpret_cast<uintptr_t>(m->d_q_start) | reinterpret_cast<uintptr_t>(m->d_kv_len) |
                          reinterpret_cast<uintptr_t>(m->d_pos) | reinterpret_cast<uintptr_t>(m->d_seq) |
                          reinterpret_cast<uintptr_t>(m->d_info);
    if ((low & 3u) || (reinterpret_cast<uintptr_t>(m->d_cells) & 7u))
        return layer_fail(KVM_EINVAL, "%s: buffers must be aligned to their elements", me);
    PointerDevice dev(m->d_past, me);
    if (dev.status() != KVM_OK) return dev.status();
    const uint64_t work = std::max<uint64_t>(m->n_rows, static_cast<uint64_t>(m->n_seq) * 4u);
    const uint64_t want = (work + kMapThreads - 1) / kMapThreads, most = 4ull * num_sms();
    map_batch_kernel<<<static_cast<uint32_t>(want < most ? (want ? want : 1) : most), kMapThreads, 0,
                       reinterpret_cast<cudaStream_t>(stream)>>>(*m);
    return layer_cuda(cudaGetLastError(), me);
}
