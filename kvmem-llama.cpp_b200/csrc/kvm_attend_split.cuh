// kvm_attend_split.cuh -- attend_split_kernel: attention for few query rows a
// sequence (decode steps, drafted tokens), bound by reading the window once.
//
// Mathematics.  With c the unsigned code of an element, o the type's offset and
// d the scale of its block of 32 (q4_0: o = 8, q5_0: 16, q8_0: 128),
//   q . k = sum_b d_b (sum_{e in b} q_e c_e) - o sum_b d_b (sum_{e in b} q_e)
//   o_e   = sum_j (p_j d_jb) c_je - o sum_j (p_j d_jb)
// so the tensor cores see the codes themselves and nothing is rounded by
// dequantizing.  A code enters as the F16 bit pattern of its integer -- the
// subnormal c * 2^-24, exact -- which costs one AND a pair of values and no
// conversion; the factor 2^24 is taken out again in F32.  The second term of
// q . k is one more product, scales (16 keys x blocks) times block sums of q
// (an F16 value and its remainder); that of o_e a second product with the
// constant -o for A.
//
// Rounding: q enters in F16, scaled by a power of two a row so that its largest
// element is near the top of the range (exact for F16 and BF16 inputs but for
// elements 2^17 below the row's largest); p and p*d are rounded to F16 (2^-11
// relative, as the output type), sums and statistics are F32; the two terms of o_e cancel
// where values are small beside their block's largest, to some 2^-18 of that.  To use F16's
// range, p is carried times 2^14 (which cancels in the quotient) and the scales
// of V times a power of two for each block of 32 dims, which brings the largest met so far to
// [1, 2): weights keep all bits down to 2^-28 of the row's largest, scales down to 2^-14 of
// the largest of the same dims.
//
// Layout.  S^T = K Q^T with 16 keys as M and 8 query rows as N, then
// O^T = V^T P^T with dims as M: the few rows fill N = 8, codes are the A operand
// straight from the rows' bytes, and P^T goes from the accumulators to the B
// operand by one 8x8 transpose a half.  Which 16 elements of a block form one
// K = 16 product is free as long as q agrees, so every lane takes the bytes of
// one word.  A warp streams its own keys (32 or 16 a step) of one KV head through its
// own ring in shared memory and keeps its own running maximum, sum and output;
// the warps of a CTA meet once a segment.  A CTA takes up to four KV heads of the
// same keys: their slices share 32-byte sectors, and read by different CTAs at
// different times they cost 1.7 times the window's bytes (961 of 569 MB over 32
// windows).  The slices come by TMA, 2D boxes of 16 rows, where those lie in one
// block and rows are multiples of 16 bytes, else by cp.async.
//
// Measured (24 query and 4 KV heads of 256).  32 requests over ragged windows of up
// to 32768 keys, q4_0: 164 us for 569 MB = 3.5 TB/s (q5_0 275, q8_0 207, F16 333 us, the last
// the bytes' own 328); 16 of up to 20001, q8_0 keys and q4_0 values: 76 us = 3.8 TB/s.  No unit
// is full: three warps a scheduler, each a chain of dependent steps, take 52 % of the issue
// slots and 29 % of the tensor pipe, whose m16n8k16 takes 8 cycles for 8 rows of N of which 6
// are used; of 49 products a 16-key step 16 are the offset's.  168 registers, 78 bytes of
// spills.  One request of 32768 keys (38 MB, in L2 when repeated): 25 us, 11 of them a
// CTA's (queries and first rows 5, steps 3, merge 2), the rest launches and the join.
// 2 requests of up to 333 keys (2 heads of 128): 10 us.  With 16 rows (two products a
// code; 255 registers, 580 bytes of spills) the time is 1.6 times that of 8.
#pragma once

#include "kvm_attend.cuh"

namespace kvm {

template <int D, int KT, int VT, int NT>
struct SplitGeom {
    using K = Slice<KT, D>;
    using V = Slice<VT, D>;
    static constexpr int kRoom = 226 * 1024;
    // shared memory of a warp with `tiles` 16-key tiles a step and `stages` steps:
    // rows; K scales as F16 and F32, V scales as F16; two barriers and a mask a step
    static constexpr int warp_bytes(int tiles, int stages) {
        return stages * tiles * 16 * (K::kStride + V::kStride) + 1024 * tiles + stages * 24;
    }
    static constexpr bool fits(int warps, int tiles, int stages) { return warps * warp_bytes(tiles, stages) + 128 <= kRoom; }
    // 32 keys a step where they fit: the step's fixed work (ring, statistics,
    // shuffles) is half of the instructions at 16 keys.  Twelve warps where the
    // registers (D / 4 a row tile for the output) and the rows allow it.  K and V have
    // barriers of their own, so that one stage is enough: K's next rows are under way
    // during the V products and the other way round.
    static constexpr int kMany = D * NT <= 256 ? 12 : 8;
    static constexpr int kTiles = fits(8, 2, 1) ? 2 : 1;                   // 16-key tiles a step
    static constexpr int kStep = 16 * kTiles;
    static constexpr int kWarps = fits(kMany, kTiles, 1) ? kMany : fits(8, kTiles, 1) ? 8 : 4;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kStages = fits(kWarps, kTiles, 3) ? 3 : fits(kWarps, kTiles, 2) ? 2 : 1;
    static constexpr int kRowsK = kStep * K::kStride, kRowsV = kStep * V::kStride;
    static constexpr int kStage = kRowsK + kRowsV;
    static constexpr int kScaleBytes = 1024 * kTiles;
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kMerge = kWarps * 8 * NT * (D + 4 + 2) * 4;
    static constexpr int kBig = ((kRing > kMerge ? kRing : kMerge) + 127) / 128 * 128;
    static constexpr int kSmem = kBig + kWarps * (kScaleBytes + kStages * 24);
};

// a / b, by a 32-bit division where a allows it (the 64-bit routine is ten times as long)
__host__ __device__ __forceinline__ unsigned long long div_small(unsigned long long a, uint32_t b) {
    return (a >> 32) == 0 ? static_cast<uint32_t>(a) / b : a / b;
}

__device__ __forceinline__ uint32_t lds32(const uint8_t *p) { return *reinterpret_cast<const uint32_t *>(p); }
__device__ __forceinline__ uint32_t lds16(const uint8_t *p) { return *reinterpret_cast<const uint16_t *>(p); }

__device__ __forceinline__ uint32_t pack_half2(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
    const __half2 h = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&h);
}

// The codes that lane (g, t) supplies of a row's block pair `p` as A operands
// of K: w[b][m] holds the two registers (k = 2t.. and k = 2t+8..) of block
// 2p + b, product m.  Elements (q4_0, q5_0): m = 0: 4t, 4t+2 | 4t+1, 4t+3;
// m = 1: the same + 16, times 16.  (q8_0, F16): m: 8t+4m, +1 | +2, +3.
template <int KT>
__device__ __forceinline__ void k_codes(const uint8_t *pair, int t, uint32_t (&w)[2][2][2]) {
    constexpr uint32_t kLo = 0x000f000fu, kHi = 0x00f000f0u;
    if constexpr (KT == KVM_TYPE_Q4_0) {
        const uint32_t x0 = __byte_perm(lds32(pair + 4 * t), lds32(pair + 4 * t + 4), 0x5432);
        const uint32_t x1 = lds32(pair + 20 + 4 * t);
        w[0][0][0] = x0 & kLo; w[0][0][1] = (x0 >> 8) & kLo;
        w[0][1][0] = x0 & kHi; w[0][1][1] = (x0 >> 8) & kHi;
        w[1][0][0] = x1 & kLo; w[1][0][1] = (x1 >> 8) & kLo;
        w[1][1][0] = x1 & kHi; w[1][1][1] = (x1 >> 8) & kHi;
    } else if constexpr (KT == KVM_TYPE_Q5_0) {
        const uint32_t h[2] = {__byte_perm(lds32(pair), lds32(pair + 4), 0x5432) >> (4 * t),
                               lds32(pair + 24) >> (4 * t)};
        const uint32_t x[2] = {__byte_perm(lds32(pair + 4 + 4 * t), lds32(pair + 8 + 4 * t), 0x5432),
                               lds32(pair + 28 + 4 * t)};
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint32_t hl = h[b], hh = h[b] >> 16;
            // bit i of the low half-word is element 4t + i's fifth bit: spread
            // bits 0, 2 (and 1, 3) to bits 4 and 20, those of +16 to 8 and 24
            w[b][0][0] = (x[b] & kLo) | (((hl & 5u) * 0x00040010u) & 0x00100010u);
            w[b][0][1] = ((x[b] >> 8) & kLo) | (((hl & 10u) * 0x00020008u) & 0x00100010u);
            w[b][1][0] = (x[b] & kHi) | (((hh & 5u) * 0x00400100u) & 0x01000100u);
            w[b][1][1] = ((x[b] >> 8) & kHi) | (((hh & 10u) * 0x00200080u) & 0x01000100u);
        }
    } else if constexpr (KT == KVM_TYPE_Q8_0) {
        const uint32_t a0 = lds32(pair + 8 * t), a1 = lds32(pair + 8 * t + 4), a2 = lds32(pair + 8 * t + 8);
        const uint32_t x[2][2] = {{__byte_perm(a0, a1, 0x5432) ^ 0x80808080u, __byte_perm(a1, a2, 0x5432) ^ 0x80808080u},
                                  {lds32(pair + 36 + 8 * t) ^ 0x80808080u, lds32(pair + 40 + 8 * t) ^ 0x80808080u}};
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                w[b][m][0] = __byte_perm(x[b][m], 0u, 0x4140);
                w[b][m][1] = __byte_perm(x[b][m], 0u, 0x4342);
            }
    } else {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint4 x = *reinterpret_cast<const uint4 *>(pair + 64 * b + 16 * t);
            w[b][0][0] = x.x; w[b][0][1] = x.y; w[b][1][0] = x.z; w[b][1][1] = x.w;
        }
    }
}

// V: lane (g, t) supplies dims of rows g and g + 8 of two M = 16 tiles of block
// b for the keys 2t, 2t+1 (x0, x1) packed in one register: r[tile][half].
// Dims (q4_0, q5_0): 2g, 2g+1 | 16+2g, 16+2g+1 (times 16); (q8_0, F16): 4g .. 4g+3.
template <int VT>
__device__ __forceinline__ void v_codes(const uint8_t *row0, const uint8_t *row1, int b, int g, uint32_t (&r)[2][2]) {
    constexpr uint32_t kLo = 0x000f000fu, kHi = 0x00f000f0u;
    constexpr int kB = Slice<VT, 64>::kBlock;
    const uint8_t *p0 = row0 + b * kB, *p1 = row1 + b * kB;
    if constexpr (VT == KVM_TYPE_Q4_0 || VT == KVM_TYPE_Q5_0) {
        const uint32_t u = lds16(p0 + kB - 16 + 2 * g) | (lds16(p1 + kB - 16 + 2 * g) << 16);
        r[0][0] = u & kLo;
        r[0][1] = (u >> 8) & kLo;
        r[1][0] = u & kHi;
        r[1][1] = (u >> 8) & kHi;
        if constexpr (VT == KVM_TYPE_Q5_0) {
            const uint32_t l = (lds16(p0 + 2) >> (2 * g)) | ((lds16(p1 + 2) >> (2 * g)) << 16);
            const uint32_t h = (lds16(p0 + 4) >> (2 * g)) | ((lds16(p1 + 4) >> (2 * g)) << 16);
            r[0][0] |= (l << 4) & 0x00100010u;
            r[0][1] |= (l << 3) & 0x00100010u;
            r[1][0] |= (h << 8) & 0x01000100u;
            r[1][1] |= (h << 7) & 0x01000100u;
        }
    } else if constexpr (VT == KVM_TYPE_Q8_0) {
        const uint32_t l = (lds16(p0 + 2 + 4 * g) | (lds16(p1 + 2 + 4 * g) << 16)) ^ 0x80808080u;
        const uint32_t h = (lds16(p0 + 4 + 4 * g) | (lds16(p1 + 4 + 4 * g) << 16)) ^ 0x80808080u;
        r[0][0] = l & 0x00ff00ffu;
        r[0][1] = (l >> 8) & 0x00ff00ffu;
        r[1][0] = h & 0x00ff00ffu;
        r[1][1] = (h >> 8) & 0x00ff00ffu;
    } else {
        const uint2 x = *reinterpret_cast<const uint2 *>(p0 + 8 * g), y = *reinterpret_cast<const uint2 *>(p1 + 8 * g);
        r[0][0] = __byte_perm(x.x, y.x, 0x5410);
        r[0][1] = __byte_perm(x.x, y.x, 0x7632);
        r[1][0] = __byte_perm(x.y, y.y, 0x5410);
        r[1][1] = __byte_perm(x.y, y.y, 0x7632);
    }
}

// Dim of block b that tile `tile`, row half `h` holds for lane g.
template <int VT>
__device__ __forceinline__ constexpr int v_dim(int b, int tile, int h, int g) {
    return 32 * b + (Slice<VT, 64>::kNibble ? 16 * tile + 2 * g + h : 4 * g + 2 * tile + h);
}

// One value of a row slice in shared memory, by its definition.
template <int T>
__device__ __forceinline__ float row_value(const uint8_t *row, int e) {
    if constexpr (T == KVM_TYPE_F16) {
        return __half2float(*reinterpret_cast<const __half *>(row + 2 * e));
    } else {
        constexpr int kB = Slice<T, 64>::kBlock;
        const uint8_t *p = row + e / 32 * kB;
        const float d = __half2float(*reinterpret_cast<const __half *>(p));
        const int i = e % 32;
        if constexpr (T == KVM_TYPE_Q8_0) return d * static_cast<float>(static_cast<int8_t>(p[2 + i]));
        const uint32_t byte = p[kB - 16 + (i & 15)];
        int c = static_cast<int>(i < 16 ? byte & 15u : byte >> 4);
        if constexpr (T == KVM_TYPE_Q5_0) c |= static_cast<int>((p[2 + i / 8] >> (i & 7)) & 1u) << 4;
        return d * static_cast<float>(c - Slice<T, 64>::kOffset);
    }
}

template <int D, int KT, int VT, int NT>
__global__ void __launch_bounds__((SplitGeom<D, KT, VT, NT>::kThreads), 1) attend_split_kernel(const __grid_constant__ AttendArgs a) {
    using G = SplitGeom<D, KT, VT, NT>;
    using SK = Slice<KT, D>;
    using SV = Slice<VT, D>;
    constexpr int NB = D / 32, W = G::kWarps, kThreads = G::kThreads, NS = G::kStages, R = 8 * NT;
    constexpr int MT = G::kTiles, kStep = G::kStep;
    // beginning a segment (its queries, the first rows, the warps' merge) counts as
    // this many steps in the shares
    const uint32_t kLead = a.whole ? 0u : kAttendSegmentSteps / MT;
    constexpr uint32_t kAll = MT == 2 ? 0xffffffffu : 0xffffu;
    constexpr bool kCodesK = KT != KVM_TYPE_F16, kCodesV = VT != KVM_TYPE_F16;
    constexpr float kNegInf = -__builtin_huge_valf(), kWeightLog = 14.0f;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int hg = static_cast<int>(a.heads_cta), hsub = warp % hg, sub = warp / hg, nsub = W / hg;
    uint8_t *ring = smem + warp * NS * G::kStage;
    uint8_t *scales = smem + G::kBig + warp * G::kScaleBytes;
    // K scales in F32 [key][8 blocks]; V scales in F16, for each 16 keys [8 blocks][a lane's four keys
    // together], 20 halves a block (its readers' and writers' banks differ)
    float *k32 = reinterpret_cast<float *>(scales);
    __half *v16 = reinterpret_cast<__half *>(scales + 512 * MT);
    constexpr int kVBlock = 20, kVTile = 8 * kVBlock;
    uint64_t *k_bar = reinterpret_cast<uint64_t *>(smem + G::kBig + W * G::kScaleBytes) + warp * NS, *v_bar = k_bar + W * NS;
    uint32_t *valid = reinterpret_cast<uint32_t *>(smem + G::kBig + W * (G::kScaleBytes + NS * 16)) + warp * NS;
    __shared__ unsigned long long s_scan[W], s_off;
    __shared__ uint32_t s_seq;

    if (lane == 0)
        for (int i = 0; i < NS; ++i) {
            mbar_init(&k_bar[i], MT);
            mbar_init(&v_bar[i], MT);
        }
    fence_mbar_init();

    // ---- this CTA's share of the line of steps
    auto units = [&](uint32_t s) -> unsigned long long {
        const AttendSeq q = attend_seq(a, s);
        const uint64_t rows = static_cast<uint64_t>(q.n_new) * a.group;
        if (q.n_new <= 0 || rows < a.min_rows || rows > a.max_rows) return 0ull;
        const uint32_t steps = max(1u, (static_cast<uint32_t>(q.keys) + kStep - 1u) / kStep);
        return ((rows + R - 1) / R) * (a.n_head_kv / hg) * (a.whole ? 1u : steps + kLead);
    };
    // inclusive sum of n over the CTA's threads; *all gets the total
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
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w < warp) before += s_scan[w];
            sum += s_scan[w];
        }
        *all = sum;
        __syncthreads();
        return x + before;
    };
    const bool once = a.n_seq <= kThreads;
    unsigned long long mine = 0, total = 0;
    for (uint32_t s = tid; s < a.n_seq; s += kThreads) mine += units(s);
    const unsigned long long upto = scan(mine, &total);
    unsigned long long share = div_small(total + gridDim.x - 1, gridDim.x);
    // a few steps a warp at least: sharing less costs more in the join than it saves
    if (!a.whole) share = max(share, static_cast<unsigned long long>(kAttendMinSteps / MT * nsub));
    const unsigned long long u0 = share * blockIdx.x;
    const unsigned long long u1 = min(u0 + share, total);
    AttendDesc *desc = reinterpret_cast<AttendDesc *>(a.work) + blockIdx.x;
    if (u0 >= total) {
        if (tid == 0) desc->parts = 0;
        return;
    }
    unsigned long long carry = 0;
    for (uint32_t base = 0; base < a.n_seq; base += kThreads) {
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
    __syncthreads();
    uint32_t seq = s_seq;
    unsigned long long off = s_off;
    bool described = false;
    uint32_t stage_at = 0, phase = 0;         // ring stage of the warp's next step
    bool lost = false;                        // a bounded wait ran out

    for (unsigned long long pos = u0; pos < u1;) {
        // ---- the segment at `pos`
        AttendSeq q = attend_seq(a, seq);
        {
            const unsigned long long n = units(seq);
            if (off >= n) {
                off = 0;
                ++seq;
                continue;
            }
        }
        const uint32_t steps = max(1u, (static_cast<uint32_t>(q.keys) + kStep - 1u) / kStep);
        const uint32_t length = a.whole ? 1u : steps + kLead;
        const uint32_t seg = static_cast<uint32_t>(div_small(off, length));
        const uint32_t at0 = static_cast<uint32_t>(off - static_cast<unsigned long long>(seg) * length);
        const uint32_t left = length - at0;
        const uint32_t take = static_cast<uint32_t>(min(static_cast<unsigned long long>(left), u1 - pos));
        // its steps: those behind the lead
        const uint32_t in0 = at0 > kLead ? at0 - kLead : 0u, in_end = a.whole ? steps : at0 + take > kLead ? at0 + take - kLead : 0u;
        const uint32_t head0 = seg % (a.n_head_kv / hg) * hg, head = head0 + hsub;
        const uint32_t first = seg / (a.n_head_kv / hg) * R;
        const uint32_t all_rows = static_cast<uint32_t>(q.n_new) * a.group;
        const uint32_t rows = min(static_cast<uint32_t>(R), all_rows - first);
        const int32_t kend = attend_limit(a, q, (first + rows - 1) / a.group);
        const int32_t kfull = attend_limit(a, q, first / a.group);      // every row sees the keys below

        // ---- the warp's steps: in0 + sub, + nsub, ...
        const uint32_t kstart = in0 * kStep;
        const uint32_t in1 = min(in_end, (static_cast<uint32_t>(kend) + kStep - 1u) / kStep);
        const int n_steps = !lost && in1 > in0 + sub ? static_cast<int>((in1 - in0 - sub + nsub - 1) / nsub) : 0;
        const int32_t *trow = a.table + seq * a.table_stride;
        const uint8_t *kbase = a.k + static_cast<uint64_t>(head) * SK::kBytes;
        const uint8_t *vbase = a.v + static_cast<uint64_t>(head) * SV::kBytes;

        // bytes between the slice and the 16-byte boundary its box starts at
        const int lead_k = a.tma ? static_cast<int>(head * SK::kBytes & 15u) : 0;
        const int lead_v = a.tma ? static_cast<int>(head * SV::kBytes & 15u) : 0;

        // TMA: lane h < MT brings the h-th 16 keys of a step, which lie in one block;
        // the block's slot is fetched while the load before is issued
        const int32_t lane_key = static_cast<int32_t>(kstart) + sub * kStep + 16 * lane;
        const int32_t x_k = static_cast<int32_t>(head * SK::kBytes / 16u * 4u), x_v = static_cast<int32_t>(head * SV::kBytes / 16u * 4u);
        auto entry = [&](int i) -> int32_t {
            const int32_t key = lane_key + i * nsub * kStep;
            return lane < MT && key < kend ? trow[attend_block(a, static_cast<uint32_t>(key))] : -1;
        };
        int32_t slot_next = a.tma ? entry(0) : -1;

        // load(i, side, stage): K (side 0), then V (side 1) of step i; K's call looks the
        // cells up for both
        int32_t cell = -1;
        auto load = [&](int i, auto side, uint32_t to, bool skip = false) {
            constexpr bool kIsV = decltype(side)::value != 0;
            using S = std::conditional_t<kIsV, SV, SK>;
            uint8_t *dst = ring + to * G::kStage + (kIsV ? G::kRowsK : 0);
            if (a.tma) {
                if constexpr (!kIsV) {
                    const int32_t slot = slot_next;
                    slot_next = entry(i + 1);
                    if (lane < MT) {
                        const int32_t key = lane_key + i * nsub * kStep, left = kend - key;
                        const bool ok = slot >= 0 && static_cast<uint32_t>(slot) < a.n_slots;
                        reinterpret_cast<uint16_t *>(valid + to)[lane] =
                            static_cast<uint16_t>(!ok ? 0u : left >= 16 ? 0xffffu : (1u << left) - 1u);
                        const uint32_t in_block = static_cast<uint32_t>(key) - attend_block(a, static_cast<uint32_t>(key)) * a.block_tokens;
                        cell = ok ? static_cast<int32_t>(slot * a.block_tokens + in_block) : -1;
                    }
                }
                if (lane < MT && !skip) {
                    uint64_t *bar = (kIsV ? v_bar : k_bar) + to;
                    if (cell >= 0) {
                        mbar_arrive_expect_tx(bar, 16 * S::kStride);
                        tma_load_2d(dst + lane * 16 * S::kStride, kIsV ? &a.map_v : &a.map_k, kIsV ? x_v : x_k, cell, bar);
                    } else {
                        mbar_arrive(bar);
                    }
                }
                return;
            }
            if constexpr (!kIsV) {
                const uint32_t key = kstart + (sub + i * nsub) * kStep + (lane & (kStep - 1));
                cell = -1;
                if (key < static_cast<uint32_t>(kend)) {
                    const uint32_t blk = attend_block(a, key);
                    const int32_t slot = trow[blk];
                    if (slot >= 0 && static_cast<uint32_t>(slot) < a.n_slots)
                        cell = static_cast<int32_t>(slot * a.block_tokens + (key - blk * a.block_tokens));
                }
                const uint32_t ok = __ballot_sync(0xffffffffu, cell >= 0) & kAll;
                if (lane == 0) valid[to] = ok;
            }
            const uint8_t *base = kIsV ? vbase : kbase;
            const uint64_t row_bytes = kIsV ? a.row_v : a.row_k;
            auto pieces = [&](auto width) {
                constexpr int V = decltype(width)::value, C = S::kBytes / V;
#pragma unroll 4
                for (int y = 0; y < (kStep * C + 31) / 32; ++y) {
                    const int x = lane + 32 * y, row = min(x / C, kStep - 1), c = x - row * C;
                    const int32_t cr = __shfl_sync(0xffffffffu, cell, row);
                    const uint8_t *src = base + (cr >= 0 ? cr * row_bytes + c * V : 0ull);
                    const uint32_t d = smem_u32(dst + row * S::kStride + c * V);
                    if (x < kStep * C) {
                        if constexpr (V == 16) cp_async16(d, src, cr >= 0 ? 16u : 0u);
                        else cp_async4(d, src, cr >= 0 ? 4u : 0u);
                    }
                }
            };
            if constexpr (S::kBytes % 16 == 0) {
                if (a.align16) {
                    pieces(std::integral_constant<int, 16>{});
                    return;
                }
            }
            pieces(std::integral_constant<int, 4>{});
        };
        constexpr std::integral_constant<int, 0> kSideK{};
        constexpr std::integral_constant<int, 1> kSideV{};
        auto arrived = [&](uint64_t *bar) -> bool {
            bool ok = true;
            if (a.tma) ok = __all_sync(0xffffffffu, mbar_wait_near(bar, phase));
            else cp_async_wait<2 * NS - 1>();
            __syncwarp();
            return ok;
        };
        // A wait of step i ran out, behind its K rows when k_read: no more loads, no result
        // but NaN, and what is under way lands before the merge takes the ring's memory.
        auto give_up = [&](int i, bool k_read) {
            lost = true;
            for (int k = 0; k <= NS && i + k < n_steps; ++k) {
                const uint32_t at = stage_at + k < NS ? stage_at + k : stage_at + k - NS, parity = stage_at + k < NS ? phase : phase ^ 1u;
                if (k_read ? k > 0 : k < NS) mbar_wait_bounded(&k_bar[at], parity);
                if (k < NS) mbar_wait_bounded(&v_bar[at], parity);
            }
            __syncwarp();
        };
        auto hidden = [&](uint8_t *rows, auto slice, uint32_t ok) {     // a box brings the bytes of hidden rows too: drop them
            using S = decltype(slice);
            for (int x = lane; x < kStep * (S::kBytes / 4); x += 32)
                if (!((ok >> (x % kStep)) & 1u)) *reinterpret_cast<uint32_t *>(rows + (x % kStep) * S::kStride + 4 * (x / kStep)) = 0u;
            fence_proxy_async_smem();
            __syncwarp();
        };

#pragma unroll 1
        for (int i = 0; i < NS; ++i) {
            const uint32_t to = stage_at + i < NS ? stage_at + i : stage_at + i - NS;
            const uint32_t skip = (static_cast<uint32_t>(i + warp) | in0 | seq | seg) == 0u ? a.skip : 0u;
            if (i < n_steps) load(i, kSideK, to, skip & KVM_ATTEND_TEST_SKIP_K);
            cp_async_commit();
            if (i < n_steps) load(i, kSideV, to, skip & KVM_ATTEND_TEST_SKIP_V);
            cp_async_commit();
        }

        // ---- q of this lane's columns: row first + nt*8 + g
        uint32_t qf[NT][NB][4];
        uint32_t qc[NT][2];
        float fac[NT][2];
        int32_t lim[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint32_t r = first + nt * 8 + g;
            const bool in = r < first + rows;
            const uint32_t tok = r / a.group;
            const uint8_t *qp = a.q.p + (static_cast<uint64_t>(q.row0) + (in ? tok : 0)) * a.q.nb_tok +
                                (static_cast<uint64_t>(head) * a.group + (in ? r % a.group : 0)) * a.q.nb_head;
            uint32_t raw[NB][4];              // the lane's 8 values a block, in order
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (a.q_vec) {
                    if constexpr (SK::kNibble) {
                        const uint2 u = *reinterpret_cast<const uint2 *>(qp + 64 * b + 8 * t);
                        const uint2 v = *reinterpret_cast<const uint2 *>(qp + 64 * b + 32 + 8 * t);
                        raw[b][0] = u.x; raw[b][1] = u.y; raw[b][2] = v.x; raw[b][3] = v.y;
                    } else {
                        const uint4 u = *reinterpret_cast<const uint4 *>(qp + 64 * b + 16 * t);
                        raw[b][0] = u.x; raw[b][1] = u.y; raw[b][2] = u.z; raw[b][3] = u.w;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int e = 32 * b + (SK::kNibble ? 4 * t + 2 * (k & 1) + 16 * (k >> 1) : 8 * t + 2 * k);
                        raw[b][k] = *reinterpret_cast<const uint16_t *>(qp + e * a.q.nb_dim) |
                                    static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(qp + (e + 1) * a.q.nb_dim)) << 16;
                    }
                }
            }
            auto value = [&](int b, int k, int i) {       // value i of pair k
                const uint32_t u = i ? raw[b][k] >> 16 : raw[b][k] & 0xffffu;
                const float v = a.q.bf16 ? __uint_as_float(u << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(u)));
                return in ? v : 0.0f;
            };
            float x[NB][4][2], top = 0.0f;    // by operand register, as k_codes lays them out
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        // nibbles: register k pairs values (k & 1) and (k & 1) + 2 of half k >> 1
                        x[b][k][i] = SK::kNibble ? value(b, (k & 2) + i, k & 1) : value(b, k, i);
                        top = fmaxf(top, fabsf(x[b][k][i]));
                    }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // largest element to [2^(9-o), 2^(10-o)), o = log2(offset): the sums of 32
            // elements times the offset stay in F16
            const int want = kCodesK ? 9 - SK::kOffsetLog : 9;
            const int e = static_cast<int>((__float_as_uint(top) >> 23) & 255u) - 127;
            // two steps: a factor of 2^(want - e) alone may be out of F32's range
            const int up = (top > 0.0f && e < 128) ? max(-126, min(126, want - e)) : 0;
            const float mul = (a.scale_log2 < 0.0f ? -1.0f : 1.0f) * __uint_as_float(static_cast<uint32_t>(up + 127) << 23);
            uint32_t hi[NB / 2 ? NB / 2 : 1], lo[NB / 2 ? NB / 2 : 1];
            float sums[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float sum = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float part = (SK::kNibble && k >= 2) ? 0.0625f : 1.0f;
                    const uint32_t h = pack_half2(x[b][k][0] * mul * part, x[b][k][1] * mul * part);
                    qf[nt][b][k] = h;
                    const float2 back = __half22float2(*reinterpret_cast<const __half2 *>(&h));
                    sum += (back.x + back.y) / part;
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sums[b] = -static_cast<float>(SK::kOffset) * sum;
            }
            qc[nt][0] = qc[nt][1] = 0;
#pragma unroll
            for (int b = 0; b < NB; b += 2) {
                hi[b / 2] = pack_half2(sums[b], sums[b + 1]);
                const float2 back = __half22float2(*reinterpret_cast<const __half2 *>(&hi[b / 2]));
                lo[b / 2] = pack_half2(sums[b] - back.x, sums[b + 1] - back.y);
                if (t == b / 2) {
                    qc[nt][0] = hi[b / 2];
                    qc[nt][1] = lo[b / 2];
                }
            }
            // columns 2t, 2t+1 of the accumulators: their factor and limit
            // not 0: a hidden key's -inf has to stay -inf
            const float f = fmaxf(fabsf(a.scale_log2) * __uint_as_float(static_cast<uint32_t>(127 - up) << 23), 1e-37f);
            const int32_t l = in ? attend_limit(a, q, static_cast<int32_t>(tok)) : kend;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fac[nt][i] = __shfl_sync(0xffffffffu, f, (2 * t + i) * 4);
                lim[nt][i] = __shfl_sync(0xffffffffu, l, (2 * t + i) * 4);
            }
        }

        float o[NT][NB][2][4], m[NT][2], l[NT][2], bias[NT][2];      // bias: kWeightLog - m, 0 while m is -inf
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = kNegInf;
            l[nt][0] = l[nt][1] = bias[nt][0] = bias[nt][1] = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nt][b][0][i] = o[nt][b][1][i] = 0.0f;
        }
        // o holds the output times 2^(vexp - 24), vexp from 15 down by block: lane (g, t) keeps that
        // of blocks 2t, 2t + 1 as the F16 pair 2^vexp and the largest scale bits it covers
        uint32_t vmul = 0x78007800u, vcap = 0x03ff03ffu;
        auto vexp = [&](int b) -> int {
            return 16 - static_cast<int>((((__shfl_sync(0xffffffffu, vcap, b / 2) >> (16 * (b & 1))) & 0xffffu) + 1u) >> 10);
        };

#pragma unroll 1
        for (int i = 0; i < n_steps; ++i) {
            const uint32_t at = stage_at;
            uint8_t *kr = ring + at * G::kStage + lead_k;
            uint8_t *vr = ring + at * G::kStage + G::kRowsK + lead_v;
            const int32_t key0 = static_cast<int32_t>(kstart) + (sub + i * nsub) * kStep;
            if (!arrived(&k_bar[at])) {
                give_up(i, false);
                break;
            }
            const uint32_t ok = valid[at] & kAll;         // 16 keys a step: the upper half is never written
            if (a.tma && ok != kAll) hidden(kr, SK{}, ok);

            // ---- K's scales, laid out for the products
            // lane (g, t) takes blocks 2t, 2t + 1 of keys g, g + 8, ...: no two lanes' banks meet
            uint32_t kd[2 * MT];              // F16 pairs: A operand of the offsets' product
            if constexpr (kCodesK) {
#pragma unroll
                for (int i8 = 0; i8 < 2 * MT; ++i8) {
                    kd[i8] = 0;
                    if (2 * t < NB) {
                        const uint8_t *p = kr + (8 * i8 + g) * SK::kStride + 2 * t * SK::kBlock;
                        kd[i8] = lds16(p) | lds16(p + SK::kBlock) << 16;
                        *reinterpret_cast<float2 *>(k32 + (8 * i8 + g) * 8 + 2 * t) =
                            __half22float2(*reinterpret_cast<const __half2 *>(&kd[i8]));
                    }
                }
            }
            __syncwarp();

            // ---- S^T = K Q^T
            float s[NT][MT][4];
            const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[nt][mt][j] = 0.0f;
                const uint8_t *row0 = kr + (16 * mt + g) * SK::kStride, *row1 = row0 + 8 * SK::kStride;
                float dk[2][NB < 4 ? 4 : NB];     // scales of keys g, g + 8
                if constexpr (kCodesK) {
#pragma unroll
                    for (int b = 0; b < NB; b += 4) {
                        *reinterpret_cast<float4 *>(&dk[0][b]) = *reinterpret_cast<const float4 *>(k32 + (16 * mt + g) * 8 + b);
                        *reinterpret_cast<float4 *>(&dk[1][b]) = *reinterpret_cast<const float4 *>(k32 + (16 * mt + g + 8) * 8 + b);
                    }
                }
#pragma unroll
                for (int p = 0; p < NB / 2; ++p) {
                    uint32_t c0[2][2][2], c1[2][2][2];
                    k_codes<KT>(row0 + p * 2 * SK::kBlock, t, c0);
                    k_codes<KT>(row1 + p * 2 * SK::kBlock, t, c1);
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const uint32_t a0[4] = {c0[b][0][0], c1[b][0][0], c0[b][0][1], c1[b][0][1]};
                        const uint32_t a1[4] = {c0[b][1][0], c1[b][1][0], c0[b][1][1], c1[b][1][1]};
                        const float d0 = dk[0][2 * p + b], d1 = dk[1][2 * p + b];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint32_t *qq = qf[nt][2 * p + b];
                            float(&sum)[4] = s[nt][mt];
                            if constexpr (kCodesK) {
                                float part[4];
                                mma_f16(part, a0, qq[0], qq[1], zero);
                                mma_f16(part, a1, qq[2], qq[3], part);
                                sum[0] = fmaf(d0, part[0], sum[0]);
                                sum[1] = fmaf(d0, part[1], sum[1]);
                                sum[2] = fmaf(d1, part[2], sum[2]);
                                sum[3] = fmaf(d1, part[3], sum[3]);
                            } else {
                                mma_f16(sum, a0, qq[0], qq[1], sum);
                                mma_f16(sum, a1, qq[2], qq[3], sum);
                            }
                        }
                    }
                }
                if constexpr (kCodesK) {
                    const uint32_t aw[4] = {kd[2 * mt], kd[2 * mt + 1], kd[2 * mt], kd[2 * mt + 1]};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float c[4];
                        mma_f16(c, aw, qc[nt][0], qc[nt][1], zero);
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[nt][mt][j] = fmaf(s[nt][mt][j], 16777216.0f, c[j]);
                    }
                }
            }

            __syncwarp();                     // every lane is done with this step's K rows
            if (i + NS < n_steps) load(i + NS, kSideK, at);
            cp_async_commit();

            // ---- softmax step
            const bool mixed = key0 + kStep > kfull || ok != kAll;
            uint32_t pb[NT][MT][2];
            float mn[NT][2];
            bool grew = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if (mixed) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int kk = 16 * mt + g + (j >> 1) * 8;
                            if (key0 + kk >= lim[nt][j & 1] || !((ok >> kk) & 1u)) s[nt][mt][j] = kNegInf;
                        }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float x = fmaxf(s[nt][0][i], s[nt][0][i + 2]);
                    if constexpr (MT == 2) x = fmaxf(x, fmaxf(s[nt][MT - 1][i], s[nt][MT - 1][i + 2]));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    mn[nt][i] = fmaxf(m[nt][i], x == kNegInf ? kNegInf : x * fac[nt][i]);
                    grew = grew || mn[nt][i] > m[nt][i];
                }
            }
            if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float f[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        f[i] = mn[nt][i] > m[nt][i] ? exp2_approx(m[nt][i] - mn[nt][i]) : 1.0f;
                        l[nt][i] *= f[i];
                        m[nt][i] = mn[nt][i];
                        bias[nt][i] = kWeightLog - (m[nt][i] == kNegInf ? kWeightLog : m[nt][i]);
                    }
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            o[nt][b][0][j] *= f[j & 1];
                            o[nt][b][1][j] *= f[j & 1];
                        }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[nt][mt][j] = exp2_approx(fmaf(s[nt][mt][j], fac[nt][j & 1], bias[nt][j & 1]));
                        l[nt][j & 1] += s[nt][mt][j];
                    }
                    pb[nt][mt][0] = transpose8(pack_half2(s[nt][mt][0], s[nt][mt][1]));
                    pb[nt][mt][1] = transpose8(pack_half2(s[nt][mt][2], s[nt][mt][3]));
                }

            // ---- V's rows and scales
            if (!arrived(&v_bar[at])) {
                give_up(i, true);
                break;
            }
            if (a.tma && ok != kAll) hidden(vr, SV{}, ok);
            bool odd_values = false;          // an infinite or NaN V value
            if constexpr (kCodesV) {
                uint32_t d[2 * MT], top = 0;  // pairs of blocks 2t, 2t + 1
#pragma unroll
                for (int i8 = 0; i8 < 2 * MT; ++i8) {
                    d[i8] = 0;
                    if (2 * t < NB) {
                        const uint8_t *p = vr + (8 * i8 + g) * SV::kStride + 2 * t * SV::kBlock;
                        d[i8] = lds16(p) | lds16(p + SV::kBlock) << 16;
                    }
                    top = __vmaxu2(top, d[i8] & 0x7fff7fffu);
                }
                // rarely: a scale beyond the range that vexp covers, or one that is not finite
                if (__any_sync(0xffffffffu, __vmaxu2(top, vcap) != vcap)) {
                    uint32_t cap = 0, mul = 0, move = 0;       // by half: new vcap, vmul; how far vexp falls
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t finite = 0;
#pragma unroll
                        for (int i8 = 0; i8 < 2 * MT; ++i8) {
                            const uint32_t size = (d[i8] >> (16 * h)) & 0x7fffu;
                            odd_values = odd_values || size >= 0x7c00u;
                            finite = max(finite, size >= 0x7c00u ? 0u : size);
                        }
#pragma unroll
                        for (int x = 4; x < 32; x *= 2) finite = max(finite, __shfl_xor_sync(0xffffffffu, finite, x));
                        const uint32_t old = (vcap >> (16 * h)) & 0xffffu, now = max(old, finite | 0x3ffu);
                        const uint32_t exponent = (now + 1u) >> 10;           // 16 - vexp
                        cap |= now << (16 * h);
                        mul |= (exponent <= 30u ? (31u - exponent) << 10 : 0x0200u) << (16 * h);       // the largest so far to [1, 2)
                        move |= (exponent - ((old + 1u) >> 10)) << (16 * h);
                    }
                    odd_values = __any_sync(0xffffffffu, odd_values);
                    vcap = cap;
                    vmul = mul;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const float f = __uint_as_float((127u - ((__shfl_sync(0xffffffffu, move, b / 2) >> (16 * (b & 1))) & 0xffffu)) << 23);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                o[nt][b][0][j] *= f;
                                o[nt][b][1][j] *= f;
                            }
                    }
                }
                if (2 * t < NB) {
#pragma unroll
                    for (int i8 = 0; i8 < 2 * MT; ++i8) {
                        const uint32_t ds = mul_half2(d[i8], vmul);
                        // key g of the half i8 & 1 of its 16: behind the pair's other key
                        __half *to = v16 + (i8 >> 1) * kVTile + 2 * t * kVBlock + (g >> 1) * 4 + (i8 & 1) * 2 + (g & 1);
                        to[0] = __ushort_as_half(static_cast<uint16_t>(ds & 0xffffu));
                        to[kVBlock] = __ushort_as_half(static_cast<uint16_t>(ds >> 16));
                    }
                }
            }
            __syncwarp();
            if constexpr (!kCodesV) {
                if (mixed) {                  // a hidden key's infinity must not meet p = 0 in a product
                    for (int x = lane; x < kStep * (D / 2); x += 32) {
                        const uint32_t u = lds32(vr + (x % kStep) * SV::kStride + (x / kStep) * 4);
                        odd_values = odd_values || (u & 0x7c00u) == 0x7c00u || (u & 0x7c000000u) == 0x7c000000u;
                    }
                    odd_values = __any_sync(0xffffffffu, odd_values);
                }
            }

            // ---- O^T += V^T P^T
            if (!odd_values) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const uint8_t *v0 = vr + (16 * mt + 2 * t) * SV::kStride;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        uint32_t x[2][2], y[2][2];
                        v_codes<VT>(v0, v0 + SV::kStride, b, g, x);
                        v_codes<VT>(v0 + 8 * SV::kStride, v0 + 9 * SV::kStride, b, g, y);
                        uint2 ds = make_uint2(0u, 0u);
                        if constexpr (kCodesV) ds = *reinterpret_cast<const uint2 *>(v16 + mt * kVTile + b * kVBlock + 4 * t);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            uint32_t b0 = pb[nt][mt][0], b1 = pb[nt][mt][1];
                            if constexpr (kCodesV) {
                                b0 = mul_half2(b0, ds.x);
                                b1 = mul_half2(b1, ds.y);
                            }
#pragma unroll
                            for (int tile = 0; tile < 2; ++tile) {
                                const uint32_t av[4] = {x[tile][0], x[tile][1], y[tile][0], y[tile][1]};
                                mma_f16(o[nt][b][tile], av, b0, b1, o[nt][b][tile]);
                                if constexpr (kCodesV) {
                                    // the constant -offset (times 16 in the high-nibble tile) * 2^-24
                                    constexpr uint32_t n0 = 0x8000u | SV::kOffset;
                                    constexpr uint32_t n1 = 0x8000u | (SV::kNibble ? 16 * SV::kOffset : SV::kOffset);
                                    const uint32_t cc = tile ? n1 * 0x10001u : n0 * 0x10001u;
                                    const uint32_t ac[4] = {cc, cc, cc, cc};
                                    mma_f16(o[nt][b][tile], ac, b0, b1, o[nt][b][tile]);
                                }
                            }
                        }
                    }
                }
            } else {
                // values that are not finite: by the definition, p = 0 leaves them out
                float unit[NB];
#pragma unroll
                for (int b = 0; b < NB; ++b) unit[b] = kCodesV ? __uint_as_float(static_cast<uint32_t>(vexp(b) - 24 + 127) << 23) : 1.0f;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll 1
                    for (int k = 0; k < 16; ++k) {
                        const uint8_t *row = vr + (16 * mt + k) * SV::kStride;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const int from = (k & 7) * 4 + t;
                            const float p0 = __shfl_sync(0xffffffffu, k < 8 ? s[nt][mt][0] : s[nt][mt][2], from);
                            const float p1 = __shfl_sync(0xffffffffu, k < 8 ? s[nt][mt][1] : s[nt][mt][3], from);
#pragma unroll
                            for (int b = 0; b < NB; ++b)
#pragma unroll
                                for (int tile = 0; tile < 2; ++tile)
#pragma unroll
                                    for (int h = 0; h < 2; ++h) {
                                        const float up = SV::kNibble && tile ? 16.0f : 1.0f;
                                        const float v = row_value<VT>(row, v_dim<VT>(b, tile, h, g)) * unit[b] * up;
                                        if (p0 != 0.0f) o[nt][b][tile][2 * h] += p0 * v;
                                        if (p1 != 0.0f) o[nt][b][tile][2 * h + 1] += p1 * v;
                                    }
                        }
                    }
            }
            __syncwarp();                     // ... and with its V rows
            if (i + NS < n_steps) load(i + NS, kSideV, at);
            cp_async_commit();
            if (++stage_at == NS) {
                stage_at = 0;
                phase ^= 1u;
            }
        }

        // ---- the warps' results together
        if (lost) {                           // no result rather than a wrong one
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) l[nt][0] = l[nt][1] = __int_as_float(0x7fc00000);
        }
        cp_async_wait<0>();
        __syncthreads();
        float *sm_m = reinterpret_cast<float *>(smem), *sm_l = sm_m + W * R, *sm_o = sm_l + W * R;
        constexpr int OS = D + 4;
        float unit[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) unit[b] = kCodesV ? __uint_as_float(static_cast<uint32_t>(24 - vexp(b) + 127) << 23) : 1.0f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x = l[nt][i];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                const int col = nt * 8 + 2 * t + i;
                if (g == 0) {
                    sm_m[warp * R + col] = m[nt][i];
                    sm_l[warp * R + col] = x;
                }
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int tile = 0; tile < 2; ++tile)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float up = SV::kNibble && tile ? 0.0625f : 1.0f;
                        sm_o[(warp * R + nt * 8 + 2 * t + (j & 1)) * OS + v_dim<VT>(b, tile, j >> 1, g)] =
                            o[nt][b][tile][j] * unit[b] * up;
                    }
        }
        __syncthreads();
        const bool starts = at0 == 0, ends = take == left, whole = starts && ends;
        // a thread a (head, row): the warps' weights; then four dims a thread
        if (tid < hg * R) {
            const int hs = tid / R, row = tid % R;
            float top = kNegInf, sum = 0.0f;
            for (int w = hs; w < W; w += hg) top = fmaxf(top, sm_m[w * R + row]);
            const float to = top == kNegInf ? 0.0f : top;
            for (int w = hs; w < W; w += hg) {
                const float f = exp2_approx(sm_m[w * R + row] - to);
                sum += f * sm_l[w * R + row];
                sm_m[w * R + row] = f;
            }
            if (whole) {              // weights that already divide by the sum
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                for (int w = hs; w < W; w += hg) sm_m[w * R + row] *= inv;
            } else {
                float *part = attend_part<D, NT>(a, 2u * blockIdx.x + (starts ? 1u : 0u), hs);
                part[row] = top;
                part[R + row] = sum;
            }
        }
        __syncthreads();
        for (int x = tid; x < hg * R * (D / 4); x += kThreads) {
            const int hr = x / (D / 4), d = (x % (D / 4)) * 4, hs = hr / R, row = hr % R;
            if (row >= static_cast<int>(rows)) continue;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int w = hs; w < W; w += hg) {
                const float f = sm_m[w * R + row];
                const float4 y = *reinterpret_cast<const float4 *>(sm_o + (w * R + row) * OS + d);
                acc.x += f * y.x;
                acc.y += f * y.y;
                acc.z += f * y.z;
                acc.w += f * y.w;
            }
            if (!whole) {
                *reinterpret_cast<float4 *>(attend_part<D, NT>(a, 2u * blockIdx.x + (starts ? 1u : 0u), hs) + 2 * R + row * D + d) = acc;
            } else {
                const uint32_t rr = first + row, tok = rr / a.group;
                uint8_t *to = const_cast<uint8_t *>(a.out.p) + (static_cast<uint64_t>(q.row0) + tok) * a.out.nb_tok +
                              (static_cast<uint64_t>(head0 + hs) * a.group + rr % a.group) * a.out.nb_head + d * a.out.nb_dim;
                store16(to, acc.x, a.out.bf16);
                store16(to + a.out.nb_dim, acc.y, a.out.bf16);
                store16(to + 2 * a.out.nb_dim, acc.z, a.out.bf16);
                store16(to + 3 * a.out.nb_dim, acc.w, a.out.bf16);
            }
        }
        if (starts && !ends && tid == 0) {
            desc->row0 = q.row0;
            desc->head = head0;
            desc->first = first;
            desc->rows = rows;
            desc->parts = 1u + static_cast<uint32_t>((pos + left - u1 + share - 1) / share);
        }
        described = described || (starts && !ends);
        fence_proxy_async_smem();             // the ring's next loads come after these reads and writes
        __syncthreads();
        pos += take;
        off += take;
    }
    if (!described && tid == 0) desc->parts = 0;
    pdl_launch_dependents();
}

// The rows of the split segments, listed by every CTA of a join: the first row
// of each segment in the order of the CTAs they start in.
constexpr int kJoinThreads = 512;
struct JoinList {
    uint32_t upto[kAttendMaxCtas];       // rows up to and with CTA c's segment
    uint32_t sums[kJoinThreads / 32], total;
};

__device__ __forceinline__ void join_list(const AttendArgs &a, uint32_t ctas, uint32_t heads, JoinList &list) {
    const AttendDesc *desc = reinterpret_cast<const AttendDesc *>(a.work);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t before = 0;
    for (uint32_t base = 0; base < ctas; base += kJoinThreads) {
        const uint32_t c = base + threadIdx.x;
        const uint32_t parts = c < ctas ? desc[c].parts : 0u, rows = c < ctas ? desc[c].rows : 0u;
        uint32_t x = parts ? rows * heads : 0u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) list.sums[warp] = x;
        __syncthreads();
        uint32_t all = 0;
        for (int w = 0; w < kJoinThreads / 32; ++w) {
            if (w < warp) x += list.sums[w];
            all += list.sums[w];
        }
        if (c < ctas) list.upto[c] = before + x;
        before += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) list.total = before;
    __syncthreads();
}

// CTA whose segment holds row x of the list, and the row in it.
__device__ __forceinline__ uint32_t join_find(const JoinList &list, uint32_t ctas, uint32_t x, uint32_t *row) {
    uint32_t c = 0;
    for (uint32_t step = 512; step; step >>= 1)
        if (c + step <= ctas && list.upto[c + step - 1] <= x) c += step;
    *row = x - (c ? list.upto[c - 1] : 0u);
    return c;
}

// One (head, row) of a split segment at a time, or, while that leaves CTAs idle, 64
// dims of it: the parts of a segment that starts in CTA c lie in slot 2c + 1, then
// 2(c + 1), 2(c + 2), ...  They are spread over groups of threads, four dims a
// thread, and added in a fixed order.  A decode step of one request is 24 rows of 148
// parts: bound by the chain of dependent reads, so a part's maximum, sum and first
// values are asked for together.
template <int D, int NT>
__global__ void __launch_bounds__(kJoinThreads) attend_join_kernel(const __grid_constant__ AttendArgs a, uint32_t ctas) {
    constexpr int R = 8 * NT, W = kJoinThreads / 32, kEarly = 6;
    static_assert(kAttendMaxCtas <= 2 * kJoinThreads, "two parts a thread");
    __shared__ float weight[2 * kJoinThreads], s_top[W], s_sum[W];
    __shared__ float4 s_acc[kJoinThreads];
    __shared__ JoinList list;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    join_list(a, ctas, a.heads_cta, list);
    const uint32_t slices = list.total * (D / 64) <= gridDim.x ? D / 64 : 1u;
    const uint32_t wide = D / 4 / slices, groups = kJoinThreads / wide;        // threads a part, parts at a time
    const uint32_t grp = tid / wide, at_dim = tid % wide;
    for (uint32_t item = blockIdx.x; item < list.total * slices; item += gridDim.x) {
        const uint32_t d = item % slices * wide + at_dim;                      // of D / 4
        uint32_t hr;
        const uint32_t c = join_find(list, ctas, item / slices, &hr);
        const AttendDesc *desc = reinterpret_cast<const AttendDesc *>(a.work) + c;
        const uint32_t parts = min(desc->parts, ctas), hs = hr / desc->rows, r = hr - hs * desc->rows;
        auto part = [&](uint32_t i) { return attend_part<D, NT>(a, i ? 2u * (c + i) : 2u * c + 1u, hs); };
        // rows start at 2 R floats behind a multiple of 16 bytes, D floats apart
        auto values = [&](uint32_t i) { return *reinterpret_cast<const float4 *>(part(i) + 2 * R + r * D + 4 * d); };
        float m[2], l[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint32_t i = tid + k * kJoinThreads;
            m[k] = i < parts ? part(i)[r] : -__builtin_huge_valf();
            l[k] = i < parts ? part(i)[R + r] : 0.0f;
        }
        float4 early[kEarly];
#pragma unroll
        for (int k = 0; k < kEarly; ++k) {
            const uint32_t i = grp + k * groups;
            early[k] = i < parts ? values(i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        float top = fmaxf(m[0], m[1]);
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (lane == 0) s_top[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, s_top[w]);
        const float ref = top == -__builtin_huge_valf() ? 0.0f : top;
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float f = exp2_approx(m[k] - ref);
            weight[tid + k * kJoinThreads] = f;
            sum += f * l[k];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto add = [&](uint32_t i, const float4 &x) {
            const float f = weight[i];
            acc.x += f * x.x;
            acc.y += f * x.y;
            acc.z += f * x.z;
            acc.w += f * x.w;
        };
#pragma unroll
        for (int k = 0; k < kEarly; ++k)
            if (grp + k * groups < parts) add(grp + k * groups, early[k]);
#pragma unroll 4
        for (uint32_t i = grp + kEarly * groups; i < parts; i += groups) add(i, values(i));
        s_acc[tid] = acc;
        __syncthreads();
        if (tid < 4 * wide) {
            float o = 0.0f, l_all = 0.0f;
            for (uint32_t k = 0; k < groups; ++k) o += reinterpret_cast<const float *>(s_acc + k * wide)[tid];
#pragma unroll
            for (int w = 0; w < W; ++w) l_all += s_sum[w];
            const uint32_t rr = desc->first + r, tok = rr / a.group, dim = item % slices * 4u * wide + tid;
            store16(const_cast<uint8_t *>(a.out.p) + (static_cast<uint64_t>(desc->row0) + tok) * a.out.nb_tok +
                        (static_cast<uint64_t>(desc->head + hs) * a.group + rr % a.group) * a.out.nb_head + dim * a.out.nb_dim,
                    l_all == 0.0f ? 0.0f : o / l_all, a.out.bf16);
        }
        __syncthreads();
    }
}

}  // namespace kvm
