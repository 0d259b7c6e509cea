// kvm_attend_tile.cuh -- attend_tile_kernel, attend_pair_kernel: attention for
// many query rows a sequence (prompt chunks, drafts).
//
// A work item is a tile of rows (token, query head of one KV head) against the
// keys they see, one key tile at a time:
//     S = Q K^T              (tcgen05, K from shared memory)
//     P = exp2(S * f - m)    -> F16 in TMEM, over S
//     O += P V               (tcgen05, P from TMEM, V from shared memory)
// K and V enter as F16 values code * d, rounded once: unlike the few-row kernel
// this one is not bound by the window's bytes, and dequantizing once for all
// rows leaves the tensor cores plain F16 operands.  V blocks that may leave F16's range
// (scales from 65536 / the largest code on, kTileWide), infinities and NaN stay out of
// the products, where a weight of 0 would make NaN of them; the epilogue adds them by
// the definition, in F32, with their own weights.  K boxes with such scales enter divided
// by the largest code, a power of two, and their columns of S are multiplied by it again.
// Q is scaled a row by a power of two (exact for 16-bit inputs but for elements 2^24
// below the row's largest), P is F16, all sums and statistics are F32.  The running
// maximum is raised only when it would grow by more than 2^8, so O in TMEM is rescaled
// rarely; P carries a factor 2^7 that cancels in the quotient, which keeps it
// below F16's top and its bits down to 2^-31 of the row's largest weight.
//
// Two shapes.
//  - One CTA (attend_tile_kernel): 128 rows, 64 keys a tile, Q in TMEM.  With D = 256
//    S 2 x 64, O 256 and Q 128 columns are all of TMEM; Q there rather than in
//    shared memory halves what S = Q K^T reads from it (A 4 KB + B 2 KB an instruction
//    otherwise, at 128 bytes a cycle).  An instruction of 128 x 64 x 16 takes 57
//    cycles, not the 32 of its rate.
//  - A pair of CTAs (attend_pair_kernel, quantized K and V of 128 or 256 dims, more
//    than 128 rows): 256 rows, 128 keys a tile by cta_group::2.  128 x 128 x 16 takes
//    65 cycles a CTA, so the pair nearly doubles the rate of S = Q K^T, and each CTA dequantizes
//    only half of every tile (64 keys of K, half of V's dims) for 256 rows.  Q is in
//    shared memory there: 2 x 128 columns of S and 256 of O fill TMEM.
//    2048 tokens behind a window of 32768 keys (24 heads of 256, q4_0): 2.29 ms by
//    single CTAs, 1.54 ms by pairs (1.54 to 1.79 ms by the card's power cap).
//
// Roles (17 warps, one CTA an SM): warps 0-7 own 128 rows (Q, softmax, epilogue),
// two threads a row with half the columns each; warps 8-11 turn raw K rows into an
// operand tile, warps 12-15 raw V rows, warp 16 issues the products.  (One thread a
// row left a single softmax warp on each scheduler, whose latencies alone took 2250
// cycles a tile.  All warps have the same 96 registers and spill 340 bytes (pairs 500)
// at 256 dims; 25 warps would have 72 and were slower.)
// Everything is double-buffered on mbarriers: S of tile j + 1 is issued before O of
// tile j, so that the softmax of one tile runs under the products of the other.
// Raw rows come through a ring a warp, 16 keys a slot, refilled as soon as a slot
// is read; the table is looked up for 32 boxes at a time.
//
// What bounds it now.  Pairs: a 128-key tile takes 4100 cycles, of which the tensor
// cores are busy for 53 %; the longest chain is a V warp's two boxes (1600 cycles
// each: 850 of conversion, the rest barriers, fences and the load's issue), with the
// softmax warps (3100) behind it.  Giving every dequantizing warp a box of K and
// one of V, half the dims each, was slower (1.67 ms).  Drafts (8 requests of 4
// tokens, 80,000 keys): 87 us against 14 for their bytes.  The time hardly depends on the
// rows: a 64-key tile costs 4000 cycles, 2100 of them a box's conversion, while six of the
// eight softmax warps sleep (their polling cost 3 us); 1.5 stalls an issue are
// instruction fetch.  F16 K and V, by single CTAs: 2.67 ms for the prompt.
//
// Operand tiles: rows of keys by 128-byte chunks of 64 dims with the 128-byte
// swizzle; K is read K-major, V from the same layout MN-major.  Which dim a
// position stands for is free as long as Q (for K) and the epilogue (for V)
// agree: q4_0 and q5_0 keep the order their nibbles fall out in (position i of
// eight holds value 0 2 1 3 4 6 5 7).
//
// The (item, key tile) pairs of the call form one line, shared evenly by the
// CTAs or pairs; an item that several share leaves its pieces' maxima, sums and
// normalised outputs for attend_tile_join_kernel: F16 values of 32 dims with a power of
// two that brings their largest to [2^14, 2^15) (one rounding as large as the output's
// own, whatever their size; F32 would take twice the workspace).
#pragma once

#include "kvm_attend_split.cuh"

namespace kvm {

constexpr int kTileRows = 128, kTileThreads = 17 * 32;      // rows of a CTA

template <int D, int KT, int VT, bool PAIR>
struct TileGeom {
    static constexpr int kRows = PAIR ? 256 : 128, kKeys = PAIR ? 128 : 64;      // an item's rows, a key tile
    using K = Slice<KT, D>;
    using V = Slice<VT, PAIR ? D / 2 : D>;                         // the dims of V that a CTA dequantizes
    static constexpr int kSlices = PAIR ? 2 : 1;                   // V slices a head
    static constexpr int kBoxesV = PAIR ? 2 : 1;                   // 16-key boxes of V a warp and tile (of K one)
    static constexpr int kOperand = 64 * D * 2;                    // a CTA's part of one K or V tile
    static constexpr int kQ = PAIR ? kTileRows * D * 2 : 0;        // Q in shared memory (else TMEM)
    static constexpr int kBoxK = kAttendBox * K::kStride, kBoxV = kAttendBox * V::kStride;
    static constexpr int kRoom = 220 * 1024 - 4 * kOperand - kQ;
    static constexpr int kFit = kRoom / (4 * (kBoxK + kBoxV));
    static constexpr int kStages = kFit > 4 ? 4 : kFit < 1 ? 1 : kFit;     // boxes a warp's raw ring holds
    static constexpr int kRaw = 4 * kOperand + kQ;                 // offset of the raw rings
    static constexpr int kBars = kRaw + 4 * kStages * (kBoxK + kBoxV);
    static constexpr int kSmem = kBars + 512 + 1024;               // barriers; alignment of the operand tiles
};

// ------------------------------------------------------------- tcgen05 PTX --
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// D[tmem] (+)= A[tmem] B[smem], F16 operands, F32 accumulator.
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
        : "memory");
}
// The same by a CTA pair: 256 rows, this CTA's and its peer's; A from TMEM or, with
// an operand descriptor, from shared memory (the same offsets in both CTAs).
__device__ __forceinline__ void tc_mma_pair(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
        : "memory");
}
__device__ __forceinline__ void tc_mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
        : "memory");
}
// Arrives on the barrier of both CTAs when the products issued so far are done.
__device__ __forceinline__ void tc_commit_pair(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(smem_u32(bar)), "h"(static_cast<uint16_t>(3))
        : "memory");
}
__device__ __forceinline__ void mbar_arrive_n(uint64_t *bar, uint32_t n) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(n) : "memory");
}
// Arrives on the barrier at the same offset in CTA `rank` of the cluster.  What the
// arrival announces lies in this SM (TMEM, shared memory) and has been completed by
// tcgen05.wait or a proxy fence before; a cluster-scope release would wait for every
// other access too, over a thousand cycles.
__device__ __forceinline__ void mbar_arrive_at(uint64_t *bar, uint32_t rank) {
    asm volatile(
        "{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, %1;\n\t"
        "mbarrier.arrive.shared::cluster.b64 _, [ra];\n\t}"
        ::"r"(smem_u32(bar)), "r"(rank)
        : "memory");
}
__device__ __forceinline__ void st_shared_at(uint32_t *p, uint32_t v, uint32_t rank) {
    asm volatile(
        "{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, %2;\n\tst.shared::cluster.u32 [ra], %1;\n\t}"
        ::"r"(smem_u32(p)), "r"(v), "r"(rank)
        : "memory");
}
__device__ __forceinline__ void st_shared_at(uint8_t *p, uint32_t v, uint32_t rank) {
    asm volatile(
        "{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, %2;\n\tst.shared::cluster.u8 [ra], %1;\n\t}"
        ::"r"(smem_u32(p)), "r"(v), "r"(rank)
        : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_ld32(uint32_t (&r)[32], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t (&r)[16], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operand descriptor: 128-byte swizzle, byte strides.
__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return static_cast<uint64_t>((addr >> 4) & 0x3fffu) | static_cast<uint64_t>((lbo >> 4) & 0x3fffu) << 16 |
           static_cast<uint64_t>((sbo >> 4) & 0x3fffu) << 32 | 1ull << 46 | 2ull << 61;
}
// Instruction descriptor: F16 x F16 -> F32.
constexpr uint32_t tc_idesc(int m, int n, bool b_mn_major) {
    return 1u << 4 | (b_mn_major ? 1u << 16 : 0u) | static_cast<uint32_t>(n / 8) << 17 | static_cast<uint32_t>(m / 16) << 24;
}

// ------------------------------------------------------------- work line --
// sum_{i < n} floor((2 i + e) / g), e >= 0, g > 0.  With e = g (e / g) + e0 and i = g k + r the
// term is e / g + 2 k + floor((2 r + e0) / g), whose last part is 0, 1 or 2: it counts how
// many of the borders g and 2 g lie at or below 2 r + e0.
__host__ __device__ inline int64_t sum_of_halves(int64_t n, int64_t e, int64_t g) {
    const int64_t e0 = e % g, turns = n / g, rest = n % g;
    const int64_t one = (g - e0 + 1) / 2, two = (2 * g - e0 + 1) / 2;      // the first r past each border
    auto part = [&](int64_t r) -> int64_t { return (r > one ? r - one : 0) + (r > two ? r - two : 0); };
    return n * (e / g) + turns * (turns - 1) * g + turns * part(g) + 2 * turns * rest + part(rest);
}

struct TileSeq {
    AttendSeq q;
    int64_t tiles;       // row tiles, 0 = not taken by this kernel
    int64_t cap;         // keys its last row sees
};

template <int ROWS>
__host__ __device__ __forceinline__ TileSeq tile_seq(const AttendArgs &a, uint32_t s) {
    TileSeq t;
    t.q = attend_seq(a, s);
    const int64_t rows = static_cast<int64_t>(t.q.n_new) * a.group;
    t.tiles = (t.q.n_new <= 0 || rows < a.min_rows || rows > a.max_rows) ? 0 : (rows + ROWS - 1) / ROWS;
    t.cap = t.q.n_new > 0 ? attend_limit(a, t.q, t.q.n_new - 1) : 0;
    return t;
}

// Key tiles of row tile i: those its last row sees, at least one.
template <int ROWS, int KEYS>
__host__ __device__ __forceinline__ int64_t tile_steps(const AttendArgs &a, const TileSeq &t, int64_t i) {
    // rows of a sequence number less than 2^31
    const int64_t last = min(static_cast<int64_t>((static_cast<uint32_t>(i + 1) * ROWS - 1u) / a.group), static_cast<int64_t>(t.q.n_new) - 1);
    const int64_t keys = attend_limit(a, t.q, static_cast<int32_t>(last));
    return max(static_cast<int64_t>(1), (keys + KEYS - 1) / KEYS);
}

// Key tiles of the first n row tiles.  Row tile i's last token is
// floor((ROWS (i + 1) - 1) / group) (the sequence's last for the last tile), so its
// count is floor((group (shift + KEYS) + ROWS (i + 1) - 1) / (KEYS group)) between the
// tiles that need one key tile and those that see `cap` keys.  ROWS is 2 KEYS, so a KEYS
// of both can be divided out first.
template <int ROWS, int KEYS>
__host__ __device__ inline int64_t tile_prefix(const AttendArgs &a, const TileSeq &t, int64_t n) {
    static_assert(ROWS == 2 * KEYS, "the sum below");
    const int64_t most = max(static_cast<int64_t>(1), (t.cap + KEYS - 1) / KEYS);
    if (!a.causal) return n * most;
    if (n <= 1) return n ? tile_steps<ROWS, KEYS>(a, t, 0) : 0;
    const int64_t g = a.group, shift = t.q.shift;
    auto first_with = [&](int64_t keys) -> int64_t {      // first tile whose last row sees at least `keys`, unclamped
        const int64_t need = g * (keys - shift - 1) - (ROWS - 1);    // ROWS i >= need
        const int64_t i = need <= 0 ? 0 : (need + ROWS - 1) / ROWS;
        return i < n ? i : n;
    };
    const int64_t ones = first_with(KEYS + 1), full = max(ones, first_with(t.cap));
    int64_t sum = ones + (n - full) * most;
    if (full > ones)
        sum += sum_of_halves(full - ones, (g * (shift + KEYS) + ROWS * ones + ROWS - 1) / KEYS, g);
    return sum;
}

// One CTA's part of one item.
struct TilePiece {
    AttendSeq q;
    uint32_t seq, head, first, rows;     // first: (token, group) row of the tile in the sequence
    int32_t in0, in1;                    // key tiles
    int32_t kend, kfull;                 // keys any row / every row sees
    bool starts, ends;
    uint32_t more;                       // CTAs behind this one that share the item
};

// Walks the pieces of a CTA; every thread of the CTA runs it alike.
template <int ROWS, int KEYS>
struct TileWalk {
    uint64_t pos, u1, share;
    uint32_t seq;
    TileSeq t;
    int64_t tile, head, in0, steps;      // where in the sequence's items

    // Position `off` of sequence s's items.
    __host__ __device__ __forceinline__ void seek(const AttendArgs &a, uint32_t s, int64_t off) {
        seq = s;
        t = tile_seq<ROWS>(a, s);
        const int64_t heads = a.n_head_kv;
        int64_t lo = 0, hi = t.tiles;    // the last tile whose items start at or before off
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) / 2;
            if (heads * tile_prefix<ROWS, KEYS>(a, t, mid) <= off) lo = mid;
            else hi = mid;
        }
        tile = lo;
        steps = tile_steps<ROWS, KEYS>(a, t, tile);
        off -= heads * tile_prefix<ROWS, KEYS>(a, t, lo);
        head = static_cast<int64_t>(div_small(static_cast<unsigned long long>(off), static_cast<uint32_t>(steps)));
        in0 = off - head * steps;
    }

    __host__ __device__ __forceinline__ bool next(const AttendArgs &a, TilePiece &p) {
        if (pos >= u1) return false;
        while (in0 == steps) {           // the next item
            in0 = 0;
            if (++head < a.n_head_kv) break;
            head = 0;
            if (++tile < t.tiles) {
                steps = tile_steps<ROWS, KEYS>(a, t, tile);
                break;
            }
            tile = 0;
            do t = tile_seq<ROWS>(a, ++seq);
            while (t.tiles == 0);        // u1 is within the line, so there is one
            steps = tile_steps<ROWS, KEYS>(a, t, 0);
        }
        const int64_t left = steps - in0;
        const int64_t take = min(left, static_cast<int64_t>(u1 - pos));
        p.q = t.q;
        p.seq = seq;
        p.head = static_cast<uint32_t>(head);
        p.first = static_cast<uint32_t>(tile) * ROWS;
        p.rows = min(static_cast<uint32_t>(ROWS), static_cast<uint32_t>(t.q.n_new) * a.group - p.first);
        p.in0 = static_cast<int32_t>(in0);
        p.kend = attend_limit(a, t.q, static_cast<int32_t>((p.first + p.rows - 1) / a.group));
        p.kfull = attend_limit(a, t.q, static_cast<int32_t>(p.first / a.group));
        p.in1 = min(static_cast<int32_t>(in0 + take), (p.kend + KEYS - 1) / KEYS);
        p.starts = in0 == 0;
        p.ends = take == left;
        p.more = p.ends ? 0u : static_cast<uint32_t>((pos + left - u1 + share - 1) / share);
        pos += take;
        in0 += take;
        return true;
    }
};

// A warp's walk in shared memory: its state is needed once a piece and would
// otherwise hold forty registers through the inner loops.
template <int ROWS, int KEYS>
struct WarpWalk {
    TileWalk<ROWS, KEYS> walk;
    TilePiece piece;
    uint32_t more;
};

// A piece's results in the workspace: maxima, sums, what 32 dims of a row were divided by,
// then rows of D halves.
template <int D, int ROWS>
__host__ __device__ constexpr uint32_t tile_part_bytes() { return ROWS * (8u + D / 8u + 2u * D); }
template <int D, int ROWS>
__device__ __forceinline__ float *tile_part_unit(uint8_t *part, uint32_t row, uint32_t dim) {
    return reinterpret_cast<float *>(part + 8 * ROWS) + row * (D / 32) + dim / 32;
}
template <int D, int ROWS>
__device__ __forceinline__ uint4 *tile_part_values(uint8_t *part, uint32_t row, uint32_t dim) {
    return reinterpret_cast<uint4 *>(part + (8 + D / 8) * ROWS + (row * D + dim) * 2);
}
template <int D, int ROWS>
__device__ __forceinline__ uint8_t *tile_part(const AttendArgs &a, uint32_t slot) {
    return a.work + kAttendMaxCtas * kAttendDescBytes + static_cast<uint64_t>(slot) * tile_part_bytes<D, ROWS>();
}

// ------------------------------------------------------------ dequantizing --
__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 h = __hfma2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b),
                              *reinterpret_cast<const __half2 *>(&c));
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Position i of eight holds value tile_order<T>(i).
template <int T>
__host__ __device__ constexpr int tile_order(int i) {
    return Slice<T, 64>::kNibble ? (i & 4) | (i & 1) << 1 | (i & 2) >> 1 : i;
}

// Magnitude bits of the first F16 scale whose block may hold values outside F16, 65536 over
// the largest code (8, 16 or 128), infinite and NaN scales among them; F16 rows: of the
// first value that is not finite.
template <int T>
constexpr uint32_t kTileWide = T == KVM_TYPE_F16 ? 0x7c00u : 0x7c00u - (static_cast<uint32_t>(Slice<T, 64>::kOffsetLog) << 10);

// The rare paths are functions of their own, one copy a kernel (KERNEL): called by all the
// kernels of a translation unit, they cost a prompt of 2048 tokens 1567 -> 1625 us.
//
// Drops from a warp's 16 raw rows what must not reach a product: hidden keys (not
// in `ok`) become zeros, and with IS_V the blocks or values that are wide (kTileWide).
template <int KERNEL, int T, int D, bool IS_V>
__device__ __noinline__ void tile_clean(uint8_t *raw, uint32_t ok, int lane) {
    using S = Slice<T, D>;
    {
        for (int x = lane; x < 16 * (S::kBytes / 4); x += 32)
            if (!((ok >> (x & 15)) & 1u)) *reinterpret_cast<uint32_t *>(raw + (x & 15) * S::kStride + (x >> 4) * 4) = 0u;
    }
    __syncwarp();
    if constexpr (IS_V) {
        constexpr int kStep = T == KVM_TYPE_F16 ? 2 : S::kBlock;      // halves to look at: every value, or the scales
        for (int x = lane; x < 16 * (S::kBytes / kStep); x += 32) {
            uint16_t *p = reinterpret_cast<uint16_t *>(raw + (x & 15) * S::kStride + (x >> 4) * kStep);
            if ((*p & 0x7fffu) >= kTileWide<T>) *p = 0;
        }
        __syncwarp();
    }
    fence_proxy_async_smem();       // before the ring's next load lands here
}

// Writes 16 keys' slices as F16 values into the operand tile; `raw` is the warp's
// 16 rows, `key0` its first row of the tile's ROWS.  An eighth of a warp takes eight
// keys' same 16-byte chunk, so reads and swizzled stores are free of bank
// conflicts.  Returns whether a scale (F16: a value) of this lane is wide.
// LOW: the values divided by 2^kOffsetLog, which keeps those of every finite scale in F16
// (exact but for values below 2^(kOffsetLog - 14)).
template <int T, int D, int ROWS, bool LOW = false>
__device__ __forceinline__ bool tile_dequant(const uint8_t *raw, uint8_t *tile, int key0, int lane) {
    uint32_t top = 0;              // largest magnitude bits of the scales
    using S = Slice<T, D>;
    const int k8 = lane & 7, quad = lane >> 3;
    auto put = [&](int key, int dim8, uint4 v) {       // dims 8 dim8 .. 8 dim8 + 7 of a key
        const int row = key0 + key;
        *reinterpret_cast<uint4 *>(tile + (dim8 >> 3) * (ROWS * 128) + row * 128 + (((dim8 & 7) ^ (row & 7)) << 4)) = v;
    };
    auto scale_at = [&](const uint8_t *p) -> uint32_t {
        const uint32_t d = lds16(p);
        top = max(top, d & 0x7fffu);
        return __byte_perm(d, 0u, 0x1010);
    };
    auto value = [&](uint32_t code, uint32_t d) -> uint32_t {
        if constexpr (LOW) code = mul_half2(code, 0x10001u * (static_cast<uint32_t>(15 - S::kOffsetLog) << 10));
        return mul_half2(code, d);
    };
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int key = 8 * half + k8;
        const uint8_t *row = raw + key * S::kStride;
        if constexpr (T == KVM_TYPE_F16) {
#pragma unroll 4
            for (int c = quad; c < D / 8; c += 4) {
                const uint4 v = *reinterpret_cast<const uint4 *>(row + 16 * c);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
                put(key, c, v);
            }
        } else if constexpr (T == KVM_TYPE_Q8_0) {
#pragma unroll 4
            for (int b = 0; b < D / 32; ++b) {
                const uint8_t *p = row + (b >> 1) * 68;
                const uint32_t d = scale_at(p + (b & 1) * 34);
                uint32_t x[2];
                if (b & 1) {
                    x[0] = lds32(p + 36 + 8 * quad);
                    x[1] = lds32(p + 40 + 8 * quad);
                } else {
                    const uint32_t w0 = lds32(p + 8 * quad), w1 = lds32(p + 8 * quad + 4), w2 = lds32(p + 8 * quad + 8);
                    x[0] = __byte_perm(w0, w1, 0x5432);
                    x[1] = __byte_perm(w1, w2, 0x5432);
                }
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t u = x[i] ^ 0x80808080u;       // 1024 + code + 128, less 1152
                    o[2 * i] = value(h2_sub(__byte_perm(u, 0x64646464u, 0x4140), 0x64806480u), d);
                    o[2 * i + 1] = value(h2_sub(__byte_perm(u, 0x64646464u, 0x4342), 0x64806480u), d);
                }
                put(key, 4 * b + quad, make_uint4(o[0], o[1], o[2], o[3]));
            }
        } else {
            // quad: block (quad >> 1) of a pair, bytes 8 h .. 8 h + 7 of its nibbles, h = quad & 1
            const int b = quad >> 1, h = quad & 1;
            constexpr int kPair = 2 * S::kBlock, kCodes = S::kBlock - 16;
            const uint32_t align = b ? 0x3210u : 0x5432u;
            // all reads first: nothing tells the compiler that the stores below do not
            // change them
            uint32_t w[D / 64][3], scale[D / 64], five[D / 64][2];
#pragma unroll
            for (int pr = 0; pr < D / 64; ++pr) {
                const uint8_t *p = row + pr * kPair;
                // q4_0: the codes start at byte 2 or 20, q5_0: 6 or 28
                const uint8_t *q = p + (b ? S::kBlock + kCodes : kCodes - 2) + 8 * h;
                scale[pr] = scale_at(p + b * S::kBlock);
                w[pr][0] = lds32(q);
                w[pr][1] = lds32(q + 4);
                w[pr][2] = lds32(q + 8);
                if constexpr (T == KVM_TYPE_Q5_0) {
                    five[pr][0] = lds16(p + b * S::kBlock + 2) >> (8 * h);
                    five[pr][1] = lds16(p + b * S::kBlock + 4) >> (8 * h);
                }
            }
#pragma unroll
            for (int pr = 0; pr < D / 64; ++pr) {
                const uint32_t d = scale[pr];
                const uint32_t x[2] = {__byte_perm(w[pr][0], w[pr][1], align), __byte_perm(w[pr][1], w[pr][2], align)};
                uint32_t lo[4], hi[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t y = x[i] >> 8;
                    uint32_t l0 = (x[i] & 0x000f000fu) | 0x64006400u, l1 = (y & 0x000f000fu) | 0x64006400u;
                    uint32_t h0 = (x[i] & 0x00f000f0u) | 0x64006400u, h1 = (y & 0x00f000f0u) | 0x64006400u;
                    if constexpr (T == KVM_TYPE_Q5_0) {
                        const uint32_t a = five[pr][0] >> (4 * i), c = five[pr][1] >> (4 * i);
                        l0 |= ((a & 5u) * 0x00040010u) & 0x00100010u;
                        l1 |= ((a & 10u) * 0x00020008u) & 0x00100010u;
                        h0 |= ((c & 5u) * 0x00400100u) & 0x01000100u;
                        h1 |= ((c & 10u) * 0x00200080u) & 0x01000100u;
                        // 1024 + n less 1040; (1024 + 16 n) / 16 less 80
                        lo[2 * i] = value(h2_sub(l0, 0x64106410u), d);
                        lo[2 * i + 1] = value(h2_sub(l1, 0x64106410u), d);
                        hi[2 * i] = value(h2_fma(h0, 0x2c002c00u, 0xd500d500u), d);
                        hi[2 * i + 1] = value(h2_fma(h1, 0x2c002c00u, 0xd500d500u), d);
                    } else {
                        // 1024 + n less 1032; (1024 + 16 n) / 16 less 72
                        lo[2 * i] = value(h2_sub(l0, 0x64086408u), d);
                        lo[2 * i + 1] = value(h2_sub(l1, 0x64086408u), d);
                        hi[2 * i] = value(h2_fma(h0, 0x2c002c00u, 0xd480d480u), d);
                        hi[2 * i + 1] = value(h2_fma(h1, 0x2c002c00u, 0xd480d480u), d);
                    }
                }
                put(key, 8 * pr + 4 * b + h, make_uint4(lo[0], lo[1], lo[2], lo[3]));
                put(key, 8 * pr + 4 * b + h + 2, make_uint4(hi[0], hi[1], hi[2], hi[3]));
            }
        }
    }
    return top >= kTileWide<T>;
}

template <int KERNEL, int T, int D, int ROWS, bool LOW>
__device__ __noinline__ void tile_dequant_again(const uint8_t *raw, uint8_t *tile, int key0, int lane) {
    tile_dequant<T, D, ROWS, LOW>(raw, tile, key0, lane);
}

// A wait ran out: results of this CTA and its peer are void from here on.
template <int KERNEL, bool PAIR>
__device__ __noinline__ void tile_say_lost(uint32_t *lost) {
    *reinterpret_cast<volatile uint32_t *>(lost) = 1u;
    if constexpr (PAIR) {
        st_shared_at(lost, 1u, (blockIdx.x & 1u) ^ 1u);
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
    } else {
        __threadfence_block();
    }
}

// Some values stay out of the tiles: the epilogues of both CTAs look for them.
template <int KERNEL, bool PAIR>
__device__ __noinline__ void tile_say_odd(uint32_t *odd) {
    *reinterpret_cast<volatile uint32_t *>(odd) = 1u;
    if constexpr (PAIR) {
        st_shared_at(odd, 1u, (blockIdx.x & 1u) ^ 1u);
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
    }
}

// A warp's raw rows did not come: its n loads under way, the ring's slots from `at` on, land
// before it goes on.
template <int KERNEL, bool PAIR>
__device__ __noinline__ void tile_abandon(uint32_t *lost, uint64_t *full, uint32_t at, uint32_t phase, uint32_t slots, int32_t n) {
    tile_say_lost<KERNEL, PAIR>(lost);
    for (uint32_t k = 0; k < slots && static_cast<int32_t>(k) < n; ++k) {
        mbar_wait_bounded(&full[at], phase);
        if (++at == slots) {
            at = 0;
            phase ^= 1u;
        }
    }
    __syncwarp();
}

// The kernel's end behind a wait that ran out: products may be under way; TMEM is freed
// behind them.
template <int KERNEL, bool PAIR>
__device__ __noinline__ void tile_finish(uint64_t *mma_done) {
    if (threadIdx.x / 32 == 16) {
        if ((threadIdx.x & 31u) == 0u && (!PAIR || (blockIdx.x & 1u) == 0u)) {
            if constexpr (PAIR) tc_commit_pair(mma_done);      // arrives in both CTAs
            else tc_commit(mma_done);
        }
        mbar_wait_bounded(mma_done, 0);
        __syncwarp();
    }
    if constexpr (PAIR) cluster_sync();
    else __syncthreads();
}

// q . k of one row and one key by the definition, in F32, from the tensors in device
// memory: for the keys whose values the tiles leave out.
template <int T, int D>
__device__ __forceinline__ float tile_score(const uint8_t *q, uint64_t nb_dim, int32_t bf16, const uint8_t *k) {
    float sum = 0.0f;
#pragma unroll 1
    for (int b = 0; b < D; b += 32)
#pragma unroll
        for (int e = b; e < b + 32; ++e) {
            const uint32_t u = *reinterpret_cast<const uint16_t *>(q + e * nb_dim);
            sum = fmaf(bf16 ? __uint_as_float(u << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(u))), row_value<T>(k, e), sum);
        }
    return sum;
}

// Adds to half `wg` of an output row, in TMEM (unnormalised, `o` the warp's columns), what the
// blocks and values that the tiles leave out of keys [lo, hi) give: weight, as the products' S
// gives it but for K's rounding, times value.  A weight that underflows leaves the value out.
// The warp looks at 32 keys at a time (up to `top`, what any of its rows sees), then every
// lane takes its row through those that have something.  1024 tokens over 8192 keys (24
// heads of 256): 0.30 ms, with one such key 0.76, with nothing else 410.
template <int KERNEL, int D, int KT, int VT>
__device__ __noinline__ void tile_add_wide(const AttendArgs &a, const TilePiece &p, const uint8_t *q, int wg, int32_t lo, int32_t hi, int32_t top,
                                           float bias, uint32_t o) {
    constexpr int kBlock = Slice<VT, 64>::kBlock, kBlocks = D / 64;
    const int lane = threadIdx.x & 31;
    float add[32 * kBlocks];
    for (int i = 0; i < 32 * kBlocks; ++i) add[i] = 0.0f;
    for (int32_t key0 = lo; key0 < top; key0 += 32) {
        int32_t cell = -1;
        uint32_t wide = 0;                     // blocks of the half, a bit each
        if (key0 + lane < top) {
            const uint32_t key = static_cast<uint32_t>(key0 + lane), blk = attend_block(a, key);
            const int32_t slot = a.table[p.seq * a.table_stride + blk];
            if (slot >= 0 && static_cast<uint32_t>(slot) < a.n_slots) {
                cell = static_cast<int32_t>(slot * a.block_tokens + (key - blk * a.block_tokens));
                const uint8_t *v = a.v + cell * a.row_v + (static_cast<uint64_t>(p.head) * 2 + wg) * (kBlocks * kBlock);
                for (int i = 0; i < kBlocks * (VT == KVM_TYPE_F16 ? 32 : 1); ++i) {
                    const int b = VT == KVM_TYPE_F16 ? i / 32 : i;
                    const uint32_t size = *reinterpret_cast<const uint16_t *>(v + (VT == KVM_TYPE_F16 ? 2 * i : i * kBlock)) & 0x7fffu;
                    wide |= (size >= kTileWide<VT> ? 1u : 0u) << b;
                }
            }
        }
        for (uint32_t any = __ballot_sync(0xffffffffu, wide != 0u); any; any &= any - 1u) {
            const int src = __ffs(any) - 1;
            const int32_t at = __shfl_sync(0xffffffffu, cell, src);
            const uint32_t blocks = __shfl_sync(0xffffffffu, wide, src);
            if (key0 + src >= hi) continue;
            const float score = tile_score<KT, D>(q, a.q.nb_dim, a.q.bf16, a.k + at * a.row_k + static_cast<uint64_t>(p.head) * Slice<KT, D>::kBytes);
            const float weight = exp2_approx(score * a.scale_log2 + bias);
            if (weight == 0.0f) continue;
            const uint8_t *v = a.v + at * a.row_v + (static_cast<uint64_t>(p.head) * 2 + wg) * (kBlocks * kBlock);
            for (int b = 0; b < kBlocks; ++b) {
                if (!((blocks >> b) & 1u)) continue;
#pragma unroll 8
                for (int i = 32 * b; i < 32 * b + 32; ++i) {
                    const float x = row_value<VT>(v, i);
                    if (VT != KVM_TYPE_F16 || !isfinite(x)) add[i] += weight * x;
                }
            }
        }
        __syncwarp();
    }
#pragma unroll 1
    for (int c = 0; c < 2 * kBlocks; ++c) {
        uint32_t x[16];
        tc_ld16(x, o + wg * 32 * kBlocks + 16 * c);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) + add[16 * c + ((i & ~7) | tile_order<VT>(i & 7))]);
        tc_st16(o + wg * 32 * kBlocks + 16 * c, x);
    }
    tc_wait_st();
}

// ------------------------------------------------------------------ kernel --
template <int D, int KT, int VT, bool PAIR>
__device__ __forceinline__ void attend_tile(const AttendArgs &a) {
    using G = TileGeom<D, KT, VT, PAIR>;
    constexpr int NS = G::kStages, kKeys = G::kKeys, kRows = G::kRows, kCtas = PAIR ? 2 : 1;
    constexpr int kKernel = 2 * VT + (PAIR ? 1 : 0);         // D and KT are alike in a translation unit
    constexpr float kNegInf = -__builtin_huge_valf(), kWeightLog = 7.0f, kSlack = 8.0f;
    constexpr uint32_t kColS = 0, kColO = 2 * kKeys, kColQ = kColO + D;       // kColQ: single CTAs only
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + G::kBars);
    uint64_t *k_full = bars, *k_free = bars + 2, *v_full = bars + 4, *v_free = bars + 6, *s_full = bars + 8, *p_full = bars + 10,
             *q_full = bars + 12, *raw_full = bars + 13, *mma_done = bars + 13 + 8 * NS;      // raw_full [8 warps][NS]
    // [4 tiles][kKeys / 16]: a bit for each hidden one of 16 keys; byte 2: their K box is LOW
    uint32_t *valid = reinterpret_cast<uint32_t *>(bars + 14 + 8 * NS);
    const uint32_t rank = PAIR ? blockIdx.x & 1u : 0u, unit = blockIdx.x / kCtas, n_units = gridDim.x / kCtas;
    __shared__ unsigned long long s_scan[kTileThreads / 32], s_off;
    __shared__ uint32_t s_seq, s_tmem, s_odd, s_lost;  // s_lost: a wait of this CTA or its peer ran out
    __shared__ float s_swap[2][2 * kTileRows];

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 4 * kCtas);
            mbar_init(&v_full[i], 4 * kCtas);
            mbar_init(&p_full[i], 8 * kCtas);
            mbar_init(&k_free[i], 1);
            mbar_init(&v_free[i], 1);
            mbar_init(&s_full[i], 1);
        }
        mbar_init(q_full, 8 * kCtas);
        // failure-path tests: one arrival more than will come, on the first rows of a K or V warp
        const int skip_k = unit == 0 && rank == 0 && (a.skip & KVM_ATTEND_TEST_SKIP_K) ? 0 : -1;
        const int skip_v = unit == 0 && rank == kCtas - 1u && (a.skip & KVM_ATTEND_TEST_SKIP_V) ? 4 * NS : -1;
        for (int i = 0; i < 8 * NS; ++i) mbar_init(&raw_full[i], i == skip_k || i == skip_v ? 2 : 1);
        mbar_init(mma_done, 1);
        s_odd = s_lost = 0;
        for (int i = 0; i < 4 * kKeys / 16; ++i) valid[i] = 0;
        fence_mbar_init();
    }
    __syncthreads();

    // ---- this CTA's share of the line of (item, key tile)
    auto units = [&](uint32_t s) -> unsigned long long {
        const TileSeq t = tile_seq<kRows>(a, s);
        return t.tiles ? static_cast<unsigned long long>(a.n_head_kv * tile_prefix<kRows, kKeys>(a, t, t.tiles)) : 0ull;
    };
    auto scan = [&](unsigned long long n, unsigned long long *all) -> unsigned long long {
        unsigned long long x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) s_scan[warp] = x;
        __syncthreads();
        unsigned long long before = 0, sum = 0;
        for (int w = 0; w < kTileThreads / 32; ++w) {
            if (w < warp) before += s_scan[w];
            sum += s_scan[w];
        }
        *all = sum;
        __syncthreads();
        return x + before;
    };
    const bool once = a.n_seq <= kTileThreads;
    unsigned long long mine = 0, total = 0;
    for (uint32_t s = tid; s < a.n_seq; s += kTileThreads) mine += units(s);
    const unsigned long long upto = scan(mine, &total);
    const unsigned long long share = max(1ull, div_small(total + n_units - 1, n_units));
    const unsigned long long u0 = share * unit, u1 = min(u0 + share, total);
    AttendDesc *desc = reinterpret_cast<AttendDesc *>(a.work) + unit;
    if (u0 >= total) {
        if (tid == 0 && rank == 0) desc->parts = 0;
        return;
    }
    unsigned long long carry = 0;
    for (uint32_t base = 0; base < a.n_seq; base += kTileThreads) {
        const uint32_t s = base + tid;
        unsigned long long n = mine, x = upto, all = total;
        if (!once) {
            n = s < a.n_seq ? units(s) : 0ull;
            x = carry + scan(n, &all);
        }
        if (n != 0 && x - n <= u0 && u0 < x) {
            s_seq = s;
            s_off = u0 - (x - n);
        }
        carry += all;
        if (carry > u0) break;
    }
    if (warp == 16) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        tc_fence_before();
    }
    __syncthreads();
    if constexpr (PAIR) cluster_sync();        // the peer's barriers and TMEM are there
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    __shared__ WarpWalk<kRows, kKeys> s_walk[kTileThreads / 32];
    WarpWalk<kRows, kKeys> &mywalk = s_walk[warp];
    const TilePiece &p = mywalk.piece;
    if (lane == 0) {
        mywalk.walk.pos = u0;
        mywalk.walk.u1 = u1;
        mywalk.walk.share = share;
        mywalk.walk.seek(a, s_seq, static_cast<int64_t>(s_off));
    }
    auto next_piece = [&]() -> bool {
        __syncwarp();                          // every lane is done with the last piece
        if (lane == 0) mywalk.more = mywalk.walk.next(a, mywalk.piece) ? 1u : 0u;
        __syncwarp();
        return mywalk.more != 0u;
    };
    // A bounded wait ran out: go on without waiting.  Whoever stores results learns of it
    // through s_lost, written before the arrival that lets the others pass.
    bool lost = false;
    auto wait = [&](uint64_t *bar, uint32_t phase) {
        if (!lost && !mbar_wait_near(bar, phase & 1u)) {
            lost = true;
            tile_say_lost<kKernel, PAIR>(&s_lost);
        }
        // together: a lane that went ahead could let the phase after this one complete
        // while another still polls for this one
        __syncwarp();
    };
    // barriers that the products wait on are the first CTA's
    auto arrive = [&](uint64_t *bar) {
        if constexpr (PAIR) mbar_arrive_at(bar, 0);
        else mbar_arrive(bar);
    };
    uint32_t j = 0;                            // running key tile of the CTA: stage j & 1, phase j >> 1

    if (warp < 8) {
        // ======== rows: Q, softmax, epilogue; thread (row, wg) has one half of S's columns and
        // of Q's and O's dims
        constexpr int kHalf = kKeys / 2;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) * 32u << 16);
        const int row = tid & 127, wg = tid >> 7;
        uint32_t swaps = 0;
        // the other thread's value of the row's pair
        auto swap = [&](float x) -> float {
            float *at = s_swap[swaps++ & 1u];
            at[wg * kTileRows + row] = x;
            asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
            return at[(wg ^ 1) * kTileRows + row];
        };
        auto vote = [&](uint64_t *bar, uint32_t n) {
            if constexpr (PAIR) mbar_arrive_at(bar, 0);
            else mbar_arrive_n(bar, n);
        };
        bool described = false;
        bool together = true;                  // every row warp is done with the pieces before this one
        while (next_piece()) {
            // Warps without a row of the piece (drafts fill one or two of the four pairs) would
            // only take the others' issue slots: they sleep on a named barrier, and the first
            // pair arrives for them.  A pair of CTAs is only used for longer requests.
            const uint32_t idle = PAIR ? 0u : 4u - min(4u, (p.rows + 31u) / 32u);
            const uint32_t votes = (warp & 3) == 0 ? 1u + idle : 1u;
            auto sleep = [&]() {
                if (idle) asm volatile("bar.sync 5, 256;" ::: "memory");
            };
            // The votes for sleeping warps let the products go over O's rows: not before those
            // warps have read there what the piece before left.
            if (!together) sleep();
            together = idle != 0u;
            if (!PAIR && static_cast<uint32_t>(warp & 3) * 32u >= p.rows) {
                j += static_cast<uint32_t>(max(0, p.in1 - p.in0));
                sleep();
                continue;
            }
            const uint32_t item_row = rank * kTileRows + row;
            const bool in = item_row < p.rows;
            const uint32_t rr = p.first + (in ? item_row : 0), tok = rr / a.group;
            const uint64_t at_tok = static_cast<uint64_t>(p.q.row0) + tok, at_head = static_cast<uint64_t>(p.head) * a.group + rr % a.group;
            const uint8_t *qp = a.q.p + at_tok * a.q.nb_tok + at_head * a.q.nb_head;
            const int32_t lim = in ? attend_limit(a, p.q, static_cast<int32_t>(tok)) : p.kend;
            // this thread's half of the row, all of it in flight at once; a piece without
            // key tiles issues no products and leaves Q alone
            constexpr int kWords = D / 4;              // of two values
            const bool work = p.in0 < p.in1;
            float fac = 0.0f;
            if (work) {
                uint32_t u[kWords];
                if (a.q_vec) {
#pragma unroll
                    for (int c = 0; c < kWords / 4; ++c) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(qp + wg * D + 16 * c);
                        u[4 * c] = v.x; u[4 * c + 1] = v.y; u[4 * c + 2] = v.z; u[4 * c + 3] = v.w;
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < kWords; ++c) {
                        const uint8_t *e = qp + (wg * (D / 2) + 2 * c) * a.q.nb_dim;
                        u[c] = *reinterpret_cast<const uint16_t *>(e) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(e + a.q.nb_dim)) << 16;
                    }
                }
                auto value = [&](int i) -> float {     // value i of the half row
                    const uint32_t w = u[i >> 1];
                    if (a.q.bf16) return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
                    return __half2float(__ushort_as_half(static_cast<uint16_t>(i & 1 ? w >> 16 : w & 0xffffu)));
                };
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < 2 * kWords; ++i) top = fmaxf(top, fabsf(value(i)));
                // the row's largest element to [2^14, 2^15): the sum of D products stays in
                // F32, 2^98 are left for K
                top = fmaxf(top, swap(top));
                const int e = static_cast<int>((__float_as_uint(top) >> 23) & 255u) - 127;
                const int up = (top > 0.0f && e < 128) ? max(-126, min(126, 14 - e)) : 0;
                const float mul = (a.scale_log2 < 0.0f ? -1.0f : 1.0f) * __uint_as_float(static_cast<uint32_t>(up + 127) << 23);
                // not 0: a hidden key's -inf has to stay -inf
                fac = fmaxf(fabsf(a.scale_log2) * __uint_as_float(static_cast<uint32_t>(127 - up) << 23), 1e-37f);
#pragma unroll
                for (int c0 = 0; c0 < D / 64; ++c0) {  // 32 dims = 16 columns at a time
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int at = 32 * c0 + 8 * (i / 4), x = 2 * (i % 4);
                        w[i] = in ? pack_half2(value(at + tile_order<KT>(x)) * mul, value(at + tile_order<KT>(x + 1)) * mul) : 0u;
                    }
                    if constexpr (PAIR) {              // K-major with the 128-byte swizzle, 64 dims a chunk
                        const int dim8 = wg * (D / 16) + 4 * c0;
                        uint8_t *to = smem + 4 * G::kOperand + row * 128;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            *reinterpret_cast<uint4 *>(to + ((dim8 + i) >> 3) * (kTileRows * 128) + ((((dim8 + i) & 7) ^ (row & 7)) << 4)) =
                                make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                    } else {
                        tc_st16(lanes + kColQ + wg * (D / 4) + 16 * c0, w);
                    }
                }
            }
            if constexpr (PAIR) fence_proxy_async_smem();
            else tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && work) vote(q_full, votes);

            float m = kNegInf, l = 0.0f;
            const uint32_t j0 = j;
            const int32_t in1 = p.in1, kfull = p.kfull;
#pragma unroll 1
            for (int32_t n = p.in0; n < in1; ++n, ++j) {
                const uint32_t st = j & 1u;
                wait(&s_full[st], j >> 1);
                // valid[] of this tile: written before k_full, which the products behind
                // s_full waited for, and not again before the tile after next's products.
                // (k_full itself may be a phase ahead here and must not be waited on.)
                tc_fence_after();
                // 32 columns at a time; a pair's thread has two such chunks and reads them twice
                uint32_t s[32];
                auto columns = [&](int c) {
                    tc_ld32(s, lanes + kColS + st * kKeys + wg * kHalf + 32 * c);
                    tc_wait_ld();
                    const uint2 word = *reinterpret_cast<const uint2 *>(valid + (kKeys / 16) * (j & 3u) + wg * (kHalf / 16) + 2 * c);
                    const int32_t key0 = n * kKeys + wg * kHalf + 32 * c;
                    if (key0 + 32 > kfull || (word.x | word.y) != 0u) {
                        if (KT != KVM_TYPE_F16 && ((word.x | word.y) >> 16) != 0u) {
                            constexpr float kUp = static_cast<float>(1 << Slice<KT, 64>::kOffsetLog);
                            const float up0 = word.x >> 16 ? kUp : 1.0f, up1 = word.y >> 16 ? kUp : 1.0f;
#pragma unroll
                            for (int i = 0; i < 32; ++i) s[i] = __float_as_uint(__uint_as_float(s[i]) * (i < 16 ? up0 : up1));
                        }
                        const uint32_t hidden = __byte_perm(word.x, word.y, 0x5410);
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (key0 + i >= lim || ((hidden >> i) & 1u)) s[i] = __float_as_uint(kNegInf);
                    }
                };
                float x = kNegInf;
#pragma unroll
                for (int c = 0; c < kHalf / 32; ++c) {
                    columns(c);
                    float t4[4] = {x, kNegInf, kNegInf, kNegInf};
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
                        t4[(i >> 1) & 3] = fmaxf(fmaxf(t4[(i >> 1) & 3], __uint_as_float(s[i])), __uint_as_float(s[i + 1]));
                    x = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
                }
                x = fmaxf(x, swap(x));
                const float mt = x == kNegInf ? kNegInf : x * fac;
                if (__any_sync(0xffffffffu, mt > m + kSlack || (m == kNegInf && mt > m))) {
                    const float mn = fmaxf(m, mt);
                    const float f = m == kNegInf ? 0.0f : exp2_approx(m - mn);
                    if (j != j0) {                     // O holds something: scale it behind the last product
                        wait(&v_free[(j - 1) & 1u], (j - 1) >> 1);
                        tc_fence_after();
#pragma unroll 1
                        for (int c = wg * (D / 32); c < (wg + 1) * (D / 32); ++c) {
                            uint32_t o[16];
                            tc_ld16(o, lanes + kColO + 16 * c);
                            tc_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(m == mn ? __uint_as_float(o[i]) : __uint_as_float(o[i]) * f);
                            tc_st16(lanes + kColO + 16 * c, o);
                        }
                        tc_wait_st();
                    }
                    l = m == mn ? l : l * f;
                    m = mn;
                }
                const float ref = m == kNegInf ? 0.0f : kWeightLog - m;
                const float2 fac2 = make_float2(fac, fac), ref2 = make_float2(ref, ref);
                float2 sum2 = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int c = 0; c < kHalf / 32; ++c) {
                    if (kHalf > 32) columns(c);
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 y = f2_fma_rn(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), fac2, ref2);
                        const float2 e = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                        sum2 = f2_add_rn(sum2, e);
                        w[i] = pack_half2(e.x, e.y);
                    }
                    // over the thread's own columns, those it has read for the last time
                    tc_st16(lanes + kColS + st * kKeys + wg * kHalf + 16 * c, w);
                }
                l += sum2.x + sum2.y;
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) vote(&p_full[st], votes);
            }
            // ---- epilogue
            const bool any = j != j0;
            if (any) {
                wait(&v_free[(j - 1) & 1u], (j - 1) >> 1);
                tc_fence_after();
                if (__any_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t *>(&s_odd) != 0))      // values the tiles left out
                    tile_add_wide<kKernel, D, KT, VT>(a, p, qp, wg, p.in0 * kKeys, in ? min(lim, p.in1 * kKeys) : 0, min(p.kend, p.in1 * kKeys),
                                                      kWeightLog - m, lanes + kColO);
            }
            if (lost || *reinterpret_cast<volatile uint32_t *>(&s_lost)) l = __int_as_float(0x7fc00000);       // no result rather than a wrong one
            l += swap(l);
            const bool whole = p.starts && p.ends;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            uint8_t *part = whole ? nullptr : tile_part<D, kRows>(a, 2u * unit + (p.starts ? 1u : 0u));
            uint8_t *op = const_cast<uint8_t *>(a.out.p) + at_tok * a.out.nb_tok + at_head * a.out.nb_head;
            if (part && wg == 0) {
                reinterpret_cast<float *>(part)[item_row] = m;
                reinterpret_cast<float *>(part)[kRows + item_row] = l;
            }
#pragma unroll 1
            for (int c = wg * (D / 64); c < (rank * kTileRows + static_cast<uint32_t>(warp & 3) * 32u < p.rows ? (wg + 1) * (D / 64) : 0); ++c) {
                uint32_t o[32];
                if (any) {
                    tc_ld32(o, lanes + kColO + 32 * c);
                    tc_wait_ld();
                }
                float y[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) y[(i & ~7) | tile_order<VT>(i & 7)] = any ? __uint_as_float(o[i]) * inv : 0.0f;
                if (part && in) {
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < 32; ++i) top = fmaxf(top, fabsf(y[i]));
                    if (!isfinite(top)) {              // the largest of the others
                        top = 0.0f;
#pragma unroll
                        for (int i = 0; i < 32; ++i) top = fmaxf(top, isfinite(y[i]) ? fabsf(y[i]) : 0.0f);
                    }
                    const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
                    const int up = min(126, 14 - e);
                    const float mul = __uint_as_float(static_cast<uint32_t>(up + 127) << 23);
                    *tile_part_unit<D, kRows>(part, item_row, 32 * c) = __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
                    uint4 *to = tile_part_values<D, kRows>(part, item_row, 32 * c);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t u[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) u[i] = pack_half2(y[8 * k + 2 * i] * mul, y[8 * k + 2 * i + 1] * mul);
                        to[k] = make_uint4(u[0], u[1], u[2], u[3]);
                    }
                } else if (!part && in) {
                    if (a.out_vec) {
                        uint4 *to = reinterpret_cast<uint4 *>(op + 64 * c);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint32_t u[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float x0 = y[8 * k + 2 * i], x1 = y[8 * k + 2 * i + 1];
                                if (a.out.bf16) {
                                    const __nv_bfloat162 b2 = __floats2bfloat162_rn(x0, x1);
                                    u[i] = *reinterpret_cast<const uint32_t *>(&b2);
                                } else {
                                    u[i] = pack_half2(x0, x1);
                                }
                            }
                            to[k] = make_uint4(u[0], u[1], u[2], u[3]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) store16(op + (32 * c + i) * a.out.nb_dim, y[i], a.out.bf16);
                    }
                }
            }
            tc_fence_before();                         // O and Q are free for the next piece's products
            if (tid == 0 && rank == 0 && p.starts && !p.ends) {
                desc->row0 = p.q.row0;
                desc->head = p.head;
                desc->first = p.first;
                desc->rows = p.rows;
                desc->parts = 1u + p.more;
            }
            described = described || (p.starts && !p.ends);
            sleep();
        }
        if (tid == 0 && rank == 0 && !described) desc->parts = 0;
    } else if (warp < 16) {
        // ======== K (warps 8-11) and V (warps 12-15): raw rows to operand tiles, a box of 16 keys at
        // a time; a tile is one box of every K warp and one or (V of a pair) two of every V warp
        const bool is_v = warp >= 12;
        const int w4 = warp & 3;
        const int raw_bytes = is_v ? G::kBoxV : G::kBoxK, boxes = is_v ? G::kBoxesV : 1;
        uint8_t *ring = smem + G::kRaw + (is_v ? 4 * NS * G::kBoxK : 0) + w4 * NS * raw_bytes;
        uint64_t *full = raw_full + (warp - 8) * NS, *tile_full = is_v ? v_full : k_full, *tile_free = is_v ? v_free : k_free;
        uint32_t in_at = 0, out_at = 0, out_phase = 0;     // ring slot of the next load, of the next box
        [[maybe_unused]] uint32_t low_tiles = 0;                            // this K warp's LOW marks in valid[], a bit a tile
        bool dead = false;                                 // rows never came: no more loads, the others are let pass
        auto pass = [&](int32_t tiles) {
            for (; tiles > 0; --tiles, ++j)
                if (lane == 0) arrive(&tile_full[j & 1u]);
        };
        // a pair's K warp also looks up the 16 keys that the peer's warp brings (their
        // visibility is wanted here too)
        constexpr int kLooks = kCtas;
        const int32_t mine = is_v ? w4 * 16 * G::kBoxesV : static_cast<int32_t>(rank) * 64 + w4 * 16;
        const int32_t theirs = is_v ? 0 : rank == 0 ? 64 : -64;
        while (next_piece()) {
            const int32_t n_tiles = max(0, p.in1 - p.in0), n_boxes = n_tiles * boxes;
            if (dead) {
                pass(n_tiles);
                continue;
            }
            const int32_t *trow = a.table + p.seq * a.table_stride;
            const uint64_t slice = is_v ? (static_cast<uint64_t>(p.head) * G::kSlices + rank) * G::V::kBytes : static_cast<uint64_t>(p.head) * G::K::kBytes;
            const int lead = a.tma ? static_cast<int>(slice & 15u) : 0;
            const int32_t x0 = static_cast<int32_t>(slice / 16u * 4u);
            uint32_t ring_ok[NS];                      // visible keys of the loads in flight
#pragma unroll
            for (int i = 0; i < NS; ++i) ring_ok[i] = 0;
            const int32_t in0 = p.in0, kend = p.kend;
            auto box_key = [&](int32_t i) -> int32_t {     // first key of box i
                return G::kBoxesV == 2 && is_v ? (in0 + (i >> 1)) * kKeys + mine + 16 * (i & 1) : (in0 + i) * kKeys + mine;
            };
            // rows and visible keys of 32 boxes, a box a lane: looking them up one by one exposed
            // the table's latency at every load (900 cycles)
            int32_t box_row = 0;
            uint32_t box_ok = 0;
            auto look = [&](int32_t i) {
                box_ok = 0;
#pragma unroll
                for (int c = 0; c < kCtas; ++c) {
                    const int32_t key0 = box_key(i) + (c ? theirs : 0), left = kend - key0;
                    const uint32_t blk = attend_block(a, static_cast<uint32_t>(max(key0, 0)));
                    const int32_t slot = i < n_boxes && left > 0 ? trow[blk] : -1;
                    const bool here = slot >= 0 && static_cast<uint32_t>(slot) < a.n_slots;
                    if (here) box_ok |= (left >= 16 ? 0xffffu : (1u << left) - 1u) << (16 * c);
                    if (c == 0 && here) box_row = static_cast<int32_t>(slot * a.block_tokens + (static_cast<uint32_t>(key0) - blk * a.block_tokens));
                }
            };
            // every lane gets the box's visible keys, a bit each (bits 16-31: those of lane 1's)
            auto load = [&](int32_t i) -> uint32_t {
                uint8_t *st = ring + in_at * raw_bytes;
                uint64_t *bar = &full[in_at];
                if (++in_at == NS) in_at = 0;
                if (a.tma) {
                    if ((i & 31) == 0) look(i + lane);
                    const uint32_t ok = __shfl_sync(0xffffffffu, box_ok, i & 31);
                    const int32_t row = __shfl_sync(0xffffffffu, box_row, i & 31);
                    if (lane == 0) {
                        if (ok & 0xffffu) {
                            mbar_arrive_expect_tx(bar, raw_bytes);
                            tma_load_2d(st, is_v ? &a.map_v : &a.map_k, x0, row, bar);
                        } else {
                            mbar_arrive(bar);
                        }
                    }
                    return ok;
                }
                const int32_t key = box_key(i) + (kLooks > 1 ? (lane & 15) + theirs * (lane >> 4) : lane & 15);
                int32_t cell = -1;
                if (key < kend) {
                    const uint32_t blk = attend_block(a, static_cast<uint32_t>(key));
                    const int32_t slot = trow[blk];
                    if (slot >= 0 && static_cast<uint32_t>(slot) < a.n_slots)
                        cell = static_cast<int32_t>(slot * a.block_tokens + (key - blk * a.block_tokens));
                }
                const uint32_t ok = __ballot_sync(0xffffffffu, cell >= 0) & (kLooks > 1 ? 0xffffffffu : 0xffffu);
                auto copy = [&](auto slice_t, const uint8_t *base, uint64_t row_bytes) {
                    using S = decltype(slice_t);
                    constexpr int C = S::kBytes / 4;
#pragma unroll 4
                    for (int y = 0; y < (kAttendBox * C + 31) / 32; ++y) {
                        const int x = lane + 32 * y, r = min(x / C, kAttendBox - 1), c = x - r * C;
                        const int32_t cr = __shfl_sync(0xffffffffu, cell, r);
                        if (x < kAttendBox * C)
                            cp_async4(smem_u32(st + r * S::kStride + c * 4), base + (cr >= 0 ? cr * row_bytes + c * 4 : 0ull), cr >= 0 ? 4u : 0u);
                    }
                };
                if (is_v) copy(typename G::V{}, a.v + slice, a.row_v);
                else copy(typename G::K{}, a.k + slice, a.row_k);
                return ok;
            };
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                if (i < n_boxes) ring_ok[i] = load(i);
                cp_async_commit();
            }
#pragma unroll 1
            for (int32_t i = 0; i < n_boxes; ++i) {
                const bool last = G::kBoxesV == 1 || !is_v || (i & 1);     // ... of its tile
                if (a.tma) {
                    const bool there = mbar_wait_near(&full[out_at], out_phase);
                    if (!__all_sync(0xffffffffu, there)) {
                        tile_abandon<kKernel, PAIR>(&s_lost, full, out_at, out_phase, NS, n_boxes - i);
                        dead = true;
                        pass(n_tiles - i / boxes);
                        break;
                    }
                } else {
                    cp_async_wait<NS - 1>();
                }
                __syncwarp();
                const uint32_t ok = ring_ok[0];
                uint8_t *raw = ring + out_at * raw_bytes + lead;
                if (++out_at == NS) {
                    out_at = 0;
                    out_phase ^= 1u;
                }
                constexpr int kVD = PAIR ? D / 2 : D;
                if ((ok & 0xffffu) != 0xffffu) {
                    if (is_v) tile_clean<kKernel, VT, kVD, false>(raw, ok & 0xffffu, lane);
                    else tile_clean<kKernel, KT, D, false>(raw, ok & 0xffffu, lane);
                }
                if (j >= 2 && (G::kBoxesV == 1 || !is_v || !(i & 1))) wait(&tile_free[j & 1u], (j >> 1) - 1u);
                uint8_t *tile = smem + (is_v ? 2 * G::kOperand : 0) + (j & 1u) * G::kOperand;
                if (is_v) {
                    const int at = w4 * 16 * G::kBoxesV + (G::kBoxesV == 2 ? 16 * (i & 1) : 0);
                    if (__any_sync(0xffffffffu, tile_dequant<VT, kVD, kKeys>(raw, tile, at, lane))) {
                        // the epilogue adds these values with their weights; the products do without them
                        tile_clean<kKernel, VT, kVD, true>(raw, ok & 0xffffu, lane);
                        tile_dequant_again<kKernel, VT, kVD, kKeys, false>(raw, tile, at, lane);
                        tile_say_odd<kKernel, PAIR>(&s_odd);
                    }
                } else {
                    const bool wide = tile_dequant<KT, D, 64>(raw, tile, w4 * 16, lane);
                    uint32_t low = 0;
                    if constexpr (KT != KVM_TYPE_F16) {
                        low = __any_sync(0xffffffffu, wide) ? 1u : 0u;
                        if (low) tile_dequant_again<kKernel, KT, D, 64, true>(raw, tile, w4 * 16, lane);
                        if (PAIR && low != ((low_tiles >> (j & 3u)) & 1u)) {       // read with the bits, so written as early
                            low_tiles ^= 1u << (j & 3u);
                            uint8_t *at = reinterpret_cast<uint8_t *>(valid + (kKeys / 16) * (j & 3u) + mine / 16) + 2;
                            if (lane < kCtas) st_shared_at(at, low, lane);
                            asm volatile("fence.acq_rel.cluster;" ::: "memory");
                        }
                    }
                    if constexpr (PAIR) {
                        if (lane < kLooks)
                            *reinterpret_cast<uint16_t *>(valid + (kKeys / 16) * (j & 3u) + (mine + theirs * lane) / 16) = static_cast<uint16_t>(~(ok >> (16 * lane)));
                    } else if (lane == 0) {
                        valid[(kKeys / 16) * (j & 3u) + mine / 16] = low << 16 | (~ok & 0xffffu);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (last) {
                    if (lane == 0) arrive(&tile_full[j & 1u]);
                    ++j;
                }
                // the box is read: its slot takes the one NS ahead
#pragma unroll
                for (int k = 0; k + 1 < NS; ++k) ring_ok[k] = ring_ok[k + 1];
                if (i + NS < n_boxes) ring_ok[NS - 1] = load(i + NS);
                cp_async_commit();
            }
            cp_async_wait<0>();
            __syncwarp();
        }
    } else if (rank == 0) {
        // ======== products, issued by one thread (of a pair: the first CTA's, for both)
        constexpr uint32_t kIdS = tc_idesc(kRows, kKeys, false), kIdO = tc_idesc(kRows, D, true);
        // descriptors of the first tiles; the others differ in the address field, which
        // no addition here carries out of
        const uint64_t k_desc = tc_desc(smem_u32(smem), 16, 1024);
        const uint64_t v_desc = tc_desc(smem_u32(smem) + 2 * G::kOperand, kKeys * 128, 1024);
        const uint64_t q_desc = tc_desc(smem_u32(smem) + 4 * G::kOperand, 16, 1024);      // pair only
        auto commit = [&](uint64_t *bar) {
            if constexpr (PAIR) tc_commit_pair(bar);
            else tc_commit(bar);
        };
        uint32_t piece = 0;
        while (next_piece()) {
            const int32_t n_tiles = max(0, p.in1 - p.in0);
            if (n_tiles == 0) continue;
            wait(q_full, piece++);
            tc_fence_after();
            const uint32_t j0 = j;
            auto qk = [&](uint32_t t) {
                wait(&k_full[t & 1u], t >> 1);
                tc_fence_after();
                const uint64_t base = k_desc + (t & 1u) * (G::kOperand / 16);
                const uint32_t to = tmem + kColS + (t & 1u) * kKeys;
                if (lane == 0) {
#pragma unroll
                    for (int s = 0; s < D / 16; ++s) {
                        const uint64_t b = base + ((s >> 2) * (64 * 128) + (s & 3) * 32) / 16;
                        if constexpr (PAIR) tc_mma_pair(to, q_desc + ((s >> 2) * (kTileRows * 128) + (s & 3) * 32) / 16, b, kIdS, s != 0);
                        else tc_mma(to, tmem + kColQ + 8 * s, b, kIdS, s != 0);
                    }
                    commit(&s_full[t & 1u]);
                    commit(&k_free[t & 1u]);
                }
                __syncwarp();
            };
            qk(j0);
            for (int32_t i = 0; i < n_tiles; ++i, ++j) {
                if (i + 1 < n_tiles) qk(j + 1);
                wait(&p_full[j & 1u], j >> 1);
                wait(&v_full[j & 1u], j >> 1);
                tc_fence_after();
                const uint64_t base = v_desc + (j & 1u) * (G::kOperand / 16);
                const uint32_t from = tmem + kColS + (j & 1u) * kKeys;
                if (lane == 0) {
#pragma unroll
                    for (int s = 0; s < kKeys / 16; ++s) {
                        // P of the first half of the keys lies at column 0, of the second at kKeys / 2
                        const uint32_t at = from + (s >= kKeys / 32 ? kKeys / 2 + 8 * (s - kKeys / 32) : 8 * s);
                        if constexpr (PAIR) tc_mma_pair(tmem + kColO, at, base + s * (2048 / 16), kIdO, i != 0 || s != 0);
                        else tc_mma(tmem + kColO, at, base + s * (2048 / 16), kIdO, i != 0 || s != 0);
                    }
                    commit(&v_free[j & 1u]);
                }
                __syncwarp();
            }
        }
    }
    __syncthreads();
    if constexpr (PAIR) cluster_sync();        // no product reads the peer's memory any more
    if (*reinterpret_cast<volatile uint32_t *>(&s_lost)) tile_finish<kKernel, PAIR>(mma_done);      // alike in a pair
    if (warp == 16) {
        tc_fence_after();
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    pdl_launch_dependents();
}

template <int D, int KT, int VT>
__global__ void __launch_bounds__(kTileThreads, 1) attend_tile_kernel(const __grid_constant__ AttendArgs a) {
    attend_tile<D, KT, VT, false>(a);
}
template <int D, int KT, int VT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTileThreads, 1) attend_pair_kernel(const __grid_constant__ AttendArgs a) {
    attend_tile<D, KT, VT, true>(a);
}

// out = sum w_i o_i / sum w_i, w_i = l_i 2^(m_i - max), over the pieces of every
// split item: a group of D / 8 threads a row, eight dims a thread.
template <int D, int ROWS>
__global__ void __launch_bounds__(kJoinThreads) attend_tile_join_kernel(const __grid_constant__ AttendArgs a, uint32_t ctas) {
    constexpr uint32_t kGroup = D / 8, kPer = kJoinThreads / kGroup;
    __shared__ JoinList list;
    pdl_wait();
    join_list(a, ctas, 1, list);
    for (uint32_t x = blockIdx.x * kPer + threadIdx.x / kGroup; x < list.total; x += gridDim.x * kPer) {
        uint32_t r;
        const uint32_t c = join_find(list, ctas, x, &r);
        const AttendDesc *desc = reinterpret_cast<const AttendDesc *>(a.work) + c;
        const uint32_t parts = min(desc->parts, ctas), d8 = threadIdx.x % kGroup;
        auto part = [&](uint32_t i) { return tile_part<D, ROWS>(a, i ? 2u * (c + i) : 2u * c + 1u); };
        // eight parts at a time, all their reads under way together, in the parts' order
        constexpr int kBatch = 8;
        float top = -__builtin_huge_valf(), sum = 0.0f, o[8] = {};
        for (uint32_t i0 = 0; i0 < parts; i0 += kBatch) {
            float m[kBatch], l[kBatch], unit[kBatch];
            uint4 v[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const bool on = i0 + k < parts;
                uint8_t *at = part(on ? i0 + k : i0);
                m[k] = on ? reinterpret_cast<const float *>(at)[r] : -__builtin_huge_valf();
                l[k] = on ? reinterpret_cast<const float *>(at)[ROWS + r] : 0.0f;
                unit[k] = *tile_part_unit<D, ROWS>(at, r, 8 * d8);
                v[k] = *tile_part_values<D, ROWS>(at, r, 8 * d8);
            }
            float next = top;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) next = fmaxf(next, m[k]);
            const float ref = next == -__builtin_huge_valf() ? 0.0f : next, f = exp2_approx(top - ref);
            top = next;
            sum *= f;
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = f == 0.0f ? 0.0f : o[k] * f;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const float w = l[k] * exp2_approx(m[k] - ref);
                const uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
                sum += w;
                if (w != 0.0f) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&u[e]));
                        o[2 * e] += w * unit[k] * y.x;
                        o[2 * e + 1] += w * unit[k] * y.y;
                    }
                }
            }
        }
        const uint32_t rr = desc->first + r, tok = rr / a.group;
        uint8_t *op = const_cast<uint8_t *>(a.out.p) + (static_cast<uint64_t>(desc->row0) + tok) * a.out.nb_tok +
                      (static_cast<uint64_t>(desc->head) * a.group + rr % a.group) * a.out.nb_head;
#pragma unroll
        for (int k = 0; k < 8; ++k) store16(op + (8 * d8 + k) * a.out.nb_dim, sum == 0.0f ? 0.0f : o[k] / sum, a.out.bf16);
    }
}

}  // namespace kvm
