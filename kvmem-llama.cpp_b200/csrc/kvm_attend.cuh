// kvm_attend.cuh -- arguments and device pieces of kvm_attend: attention of a
// step's queries over one layer's window of ggml rows.
//
//   out[r] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q_r . k_j - max)
//
// over the keys j that row r sees.  k and v stay in their blocks of 32 values
// (code * d, d the block's f16 scale); codes enter the tensor cores as exact
// small integers and the scales are applied outside the products.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kvm_internal.cuh"
#include "kvm_quant.cuh"

namespace kvm {

// One activation tensor of an attend call (kvm_rows, 16-bit types).
struct AttendRows {
    const uint8_t *p;
    uint64_t nb_dim, nb_head, nb_tok;
    int32_t bf16;              // 1 = BF16, 0 = F16
};

struct AttendArgs {
    const uint8_t *k, *v;      // one layer's cache
    uint64_t row_k, row_v;     // bytes of a cache row (all heads)
    const int32_t *table;
    uint64_t table_stride;     // entries between two sequences' rows
    uint32_t table_cols;
    const int32_t *q_start;    // [n_seq + 1]
    const int32_t *kv_len;     // [n_seq]
    uint32_t n_seq, n_rows, n_head_kv, group, block_tokens, n_slots;
    uint32_t block_shift;      // log2(block_tokens), 32 when that is no power of two
    float scale_log2;          // scale * log2(e)
    uint32_t causal;
    AttendRows q, out;
    uint8_t *work;             // split descriptors, then partial results
    uint32_t align16;          // cache bases and row bytes are multiples of 16
    uint32_t tma;              // the cache's rows come through map_k, map_v (steps lie in one block)
    uint32_t q_vec, out_vec;   // contiguous heads, 16-byte aligned
    uint32_t heads_cta;        // KV heads that a CTA takes together: 1, 2 or 4
    uint32_t whole;            // split kernel: no segment is shared (all are short), so nothing is joined
    uint32_t max_keys;         // keys that the table's columns can hold, at most 2^31 - 1
    uint32_t skip;             // the KVM_ATTEND_TEST_SKIP flags
    uint32_t min_rows, max_rows;   // query rows (tokens * group) a sequence needs to be taken by this launch
    CUtensorMap map_k, map_v;      // [cells][row bytes / 4] of 32-bit words
};

// Tensor map of one side of the cache: rows of 32-bit words, boxes of
// box_rows rows by box_bytes.  False when the driver cannot make it.
bool attend_map(CUtensorMap *map, const void *base, uint64_t row_bytes, const AttendArgs &a, uint32_t box_bytes, uint32_t box_rows);

// Keys of a request at most: a step or tile may reach some thousand keys past the
// last one, and their numbers are 32-bit.
constexpr int64_t kAttendMostKeys = 0x7fff0000;

// A sequence as the kernels see it; nothing read from device memory is trusted
// to stay inside the tables.
struct AttendSeq {
    int32_t row0;              // first row of q / out
    int32_t n_new;             // rows of this sequence inside [0, n_rows)
    int32_t shift;             // causal: row i sees keys below shift + i + 1
    int32_t keys;              // keys held by the table
};

__host__ __device__ __forceinline__ AttendSeq attend_seq(const AttendArgs &a, uint32_t s) {
    AttendSeq q;
    const int64_t lo = a.q_start[s], hi = a.q_start[s + 1];
    const int64_t kv = max(a.kv_len[s], 0);
    const int64_t cap = static_cast<int64_t>(a.table_cols) * a.block_tokens;
    const int64_t n = hi - lo;
    q.row0 = static_cast<int32_t>(lo);
    q.n_new = (lo < 0 || n <= 0 || lo >= a.n_rows)
                  ? 0 : static_cast<int32_t>(min(n, static_cast<int64_t>(a.n_rows) - lo));
    q.shift = static_cast<int32_t>(max(kv - n, static_cast<int64_t>(-0x40000000)));
    q.keys = static_cast<int32_t>(min(kv, min(cap, kAttendMostKeys)));
    return q;
}

// Keys that row token i of the sequence sees.
__host__ __device__ __forceinline__ int32_t attend_limit(const AttendArgs &a, const AttendSeq &q, int32_t i) {
    if (!a.causal) return q.keys;
    return max(0, min(q.keys, static_cast<int32_t>(min(static_cast<int64_t>(q.shift) + i + 1,
                                                       kAttendMostKeys))));
}

// Block of a key.
__device__ __forceinline__ uint32_t attend_block(const AttendArgs &a, uint32_t key) {
    return a.block_shift < 32u ? key >> a.block_shift : key / a.block_tokens;
}

__device__ __forceinline__ void store16(uint8_t *p, float x, int32_t bf16) {
    *reinterpret_cast<uint16_t *>(p) = bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x))
                                            : __half_as_ushort(__float2half_rn(x));
}

// D += A B on f16 operands with F32 accumulation, A 16x16, B 16x8.
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                        const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]),
                   "f"(c[2]), "f"(c[3]));
}

// Transpose of an 8x8 matrix of 16-bit values held two a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Bounded wait on an mbarrier phase for the short waits of a pipeline: polls
// without a suspend hint, and looks at the clock only once in a while.
__device__ __forceinline__ bool mbar_wait_near(uint64_t *bar, uint32_t parity) {
    uint64_t t0 = 0;
    for (uint32_t i = 0;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 1023u) == 1023u) {
            const uint64_t now = global_timer_ns();
            if (t0 == 0) t0 = now;
            else if (now - t0 > kWaitLimitNs) return false;
        }
    }
}

// ------------------------------------------------------- split bookkeeping --
// The keys of every (sequence, row tile, KV heads) are cut into steps of 16 or 32;
// all steps of the call form one line that the CTAs share evenly, so ragged
// batches balance without the host knowing a length.  A segment that one CTA
// holds whole is written to `out`; one that several CTAs share leaves partial
// results (max, sum, unnormalised output in F32) that attend_join_kernel adds
// in CTA order.
constexpr int kAttendBox = 16;                // rows of a TMA box
constexpr int kAttendMinSteps = 4;            // steps of 16 keys that a warp takes at least
constexpr int kAttendSegmentSteps = 24;       // steps of 16 keys that beginning a segment is worth
constexpr int kAttendWholeSteps = 4;          // steps of a warp up to which a short window is not cut
constexpr uint32_t kAttendMaxCtas = 592;      // descriptors in the workspace
constexpr uint32_t kAttendDescBytes = 32;
struct AttendDesc {                           // segment that starts in CTA c and goes on in c + 1 ...
    uint32_t parts;                           // 0 = none
    int32_t row0;                             // first token row of the tile
    uint32_t head;                            // KV head
    uint32_t first;                           // first (token, group) row of the tile in the sequence
    uint32_t rows;                            // rows of the tile
    uint32_t pad[3];
};
static_assert(sizeof(AttendDesc) == kAttendDescBytes, "AttendDesc");

// Partial results of one slot: for every head of the CTA its R maxima, R sums
// and R rows of D.
template <int D, int NT>
__host__ __device__ constexpr uint32_t attend_part_floats() { return 8u * NT * (D + 2u); }

template <int D, int NT>
__device__ __forceinline__ float *attend_part(const AttendArgs &a, uint32_t slot, uint32_t head) {
    return reinterpret_cast<float *>(a.work + kAttendMaxCtas * kAttendDescBytes) +
           (static_cast<uint64_t>(slot) * a.heads_cta + head) * attend_part_floats<D, NT>();
}

// Box of `map` at (x words, y row) to shared memory, completing on `bar`.
__device__ __forceinline__ void tma_load_2d(void *dst, const CUtensorMap *map, int32_t x, int32_t y, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}

// ------------------------------------------------------------ block codes --
// Geometry of a head's slice of a row, by cache type.
template <int T, int D>
struct Slice {
    static constexpr int kBlock = T == KVM_TYPE_F16 ? 64 : block_bytes(T);
    static constexpr int kBytes = D / 32 * kBlock;
    // a head's slice starts at a multiple of kBytes: up to this many bytes behind
    // the last 16-byte boundary
    static constexpr int kLead = kBytes % 16 == 0 ? 0 : kBytes % 8 == 0 ? 8 : 12;
    // shared-memory stride: the slice with its lead, as an odd multiple of 16
    // bytes, so that eight rows' words fall into different banks
    static constexpr int kStride = ((kBytes + kLead + 15) / 16 | 1) * 16;
    static constexpr bool kNibble = T == KVM_TYPE_Q4_0 || T == KVM_TYPE_Q5_0;
    // codes are stored unsigned; the value is (code - kOffset) * d
    static constexpr int kOffset = T == KVM_TYPE_Q4_0 ? 8 : T == KVM_TYPE_Q5_0 ? 16 : T == KVM_TYPE_Q8_0 ? 128 : 0;
    static constexpr int kOffsetLog = T == KVM_TYPE_Q4_0 ? 3 : T == KVM_TYPE_Q5_0 ? 4 : 7;
};

}  // namespace kvm
