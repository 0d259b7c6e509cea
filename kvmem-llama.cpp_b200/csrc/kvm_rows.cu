// kvm_rows.cu -- kvm_write_rows and kvm_read_rows: rows of values into and out
// of the cells of a cache, as ggml blocks.
//
// Write: the quantizers' definition in 32 bits with IEEE operations and no
// contraction (kvm_quant.cuh has the formulas), so the bytes are those of
// ggml's quantize_row_*_ref and of the stage-in.  Read: code * scale, exact in
// F32, rounded once to the output's type.
//
// Both are HBM- or latency-bound streams over 32-value blocks.  Write: a thread a
// block -- the block's maximum and its codes need no exchange -- with the values
// loaded as 16-byte vectors; the 18- to 34-byte blocks of a warp are collected in
// shared memory and leave as words, two blocks (always a whole number of words)
// at a time.  Read: a thread 16 values, two 16-byte stores.
//
// 8191 rows of 4 heads of 256 on both sides (q8_0 keys, q4_0 values), F16 in and BF16 out:
// 26 us to write and read them, 94 MB = 3.6 TB/s, over tensors larger than L2 together (22 us
// where a graph repeats one call, whose 94 MB stay in L2); a copy of those bytes takes 14.
// Issue slots are 60 % busy, with 20 to 35 % of the cycles in waits for the loads.  64 rows:
// 2.3 us each.  Types as template arguments and divisions as products took the repeated call
// from 33 us to 24, 64 instead of 74 registers (four CTAs an SM) to 22.  F16 cache
// rows move in 2-byte accesses: 144 us for 8191.
#include <cuda_bf16.h>

#include "kvm_layer.cuh"

namespace kvm {
namespace {

constexpr int kRowsThreads = 256;

struct RowsSide {
    uint8_t *cache;
    uint8_t *act;                  // source rows (write) or destination rows (read)
    uint64_t nb_dim, nb_head, nb_tok;
    uint64_t row_bytes;
    int32_t cache_type;
    uint32_t on;
};

// n / d for n < 2^31 as a product: m = floor(2^32 (2^s - d) / d) + 1, s = ceil(log2 d)
// (Granlund and Montgomery, Division by invariant integers using multiplication).
struct Divide {
    uint32_t m, s, d;
    static Divide by(uint32_t d) {
        uint32_t s = 0;
        while ((1ull << s) < d) ++s;
        return {static_cast<uint32_t>(((1ull << 32) * ((1ull << s) - d)) / d + 1u), s, d};
    }
    __device__ __forceinline__ uint32_t operator()(uint64_t n) const {
        if (n >> 31) return static_cast<uint32_t>(n / d);
        const uint32_t x = static_cast<uint32_t>(n);
        return (__umulhi(m, x) + x) >> s;
    }
};

struct RowsArgs {
    RowsSide side[2];
    const int64_t *cells;
    int64_t n_cells;
    uint32_t n, blocks, head_blocks;       // blocks of 32 a row, a head
    Divide row, head;              // by the units (blocks, or halves of them) of a row, by head_blocks
};

template <int TYPE>
__device__ __forceinline__ float act_load(const uint8_t *p) {
    if constexpr (TYPE == KVM_TYPE_F32) return *reinterpret_cast<const float *>(p);
    else if constexpr (TYPE == KVM_TYPE_F16) return __half2float(*reinterpret_cast<const __half *>(p));
    else return __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(p)) << 16);
}

template <int TYPE>
__device__ __forceinline__ void act_store(uint8_t *p, float x) {
    if constexpr (TYPE == KVM_TYPE_F32) *reinterpret_cast<float *>(p) = x;
    else if constexpr (TYPE == KVM_TYPE_F16) *reinterpret_cast<__half *>(p) = __float2half_rn(x);
    else *reinterpret_cast<__nv_bfloat16 *>(p) = __float2bfloat16_rn(x);
}

template <int TYPE>
__device__ __forceinline__ uint32_t act_pack(float x, float y) {
    if constexpr (TYPE == KVM_TYPE_F16) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

// Byte offset of block b's first value in a row of heads.
__device__ __forceinline__ uint64_t block_offset(const RowsArgs &a, const RowsSide &s, uint32_t b) {
    const uint32_t h = a.head(b);
    return h * s.nb_head + (b - h * a.head_blocks) * 32u * s.nb_dim;
}

// One block of 32 values to ggml bytes, in order.
template <int CT>
__device__ __forceinline__ void write_block(const float (&x)[32], uint8_t *dst) {
    if constexpr (CT == KVM_TYPE_F16) {
#pragma unroll
        for (int i = 0; i < 32; ++i) st_u16(dst + 2 * i, f16_bits(x[i]));
        return;
    }
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) amax = fmaxf(amax, fabsf(x[i]));
    if constexpr (CT == KVM_TYPE_Q8_0) {
        const float d = div127(amax), id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
        st_u16(dst, f16_bits(d));
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t lo = static_cast<uint32_t>(round_half_away(__fmul_rn(x[2 * i], id))) & 255u;
            const uint32_t hi = static_cast<uint32_t>(round_half_away(__fmul_rn(x[2 * i + 1], id))) & 255u;
            st_u16(dst + 2 + 2 * i, lo | hi << 8);
        }
        return;
    }
    float vmax = 0.0f;                       // the first value of the largest magnitude
#pragma unroll
    for (int i = 31; i >= 0; --i) vmax = fabsf(x[i]) == amax ? x[i] : vmax;
    vmax = __fadd_rn(vmax, 0.0f);            // a block of zeros: +0, whatever the first one's sign
    constexpr bool q5 = CT == KVM_TYPE_Q5_0;
    const float d = __fmul_rn(vmax, q5 ? -0.0625f : -0.125f), id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
    const float off = q5 ? 16.5f : 8.5f;
    const int top = q5 ? 31 : 15;
    st_u16(dst, f16_bits(d));
    uint32_t fifth = 0;
    uint8_t *qs = dst + (q5 ? 6 : 2);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t c[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {        // values 2i, 2i+1, and their partners 16 further on
            const int e = 2 * i + (k & 1) + (k >> 1) * 16;
            c[k] = static_cast<uint32_t>(min(top, __float2int_rz(__fadd_rn(__fmul_rn(x[e], id), off))));
            if (q5) fifth |= ((c[k] >> 4) & 1u) << e;
        }
        st_u16(qs + 2 * i, (c[0] & 15u) | (c[2] & 15u) << 4 | (c[1] & 15u) << 8 | (c[3] & 15u) << 12);
    }
    if (q5) {
        st_u16(dst + 2, fifth & 0xffffu);
        st_u16(dst + 4, fifth >> 16);
    }
}

// A thread a block; blocks of a row are neighbours.
template <int TYPE, bool VEC, int CT>
__device__ __forceinline__ void write_side(const RowsArgs &a, const RowsSide &s, uint8_t *stage) {
    constexpr int bb = block_bytes(CT);
    const int lane = threadIdx.x & 31;
    uint8_t *mine = stage + (threadIdx.x & ~31) * kBlockBytesQ8;
    // pairs of blocks lie in one row and start at a word: the word path
    const bool words = CT != KVM_TYPE_F16 && a.blocks % 2u == 0;
    const uint64_t all = static_cast<uint64_t>(a.n) * a.blocks;
    for (uint64_t i0 = blockIdx.x * static_cast<uint64_t>(kRowsThreads) + (threadIdx.x & ~31); i0 < all;
         i0 += static_cast<uint64_t>(gridDim.x) * kRowsThreads) {
        const uint64_t i = i0 + lane;
        const uint32_t row = a.row(i), b = static_cast<uint32_t>(i - static_cast<uint64_t>(row) * a.blocks);
        const int64_t cell = i < all ? a.cells[row] : -1;
        const bool on = cell >= 0 && cell < a.n_cells;
        uint8_t *dst = on ? s.cache + static_cast<uint64_t>(cell) * s.row_bytes + static_cast<uint64_t>(b) * bb : nullptr;
        if (on) {
            const uint8_t *src = s.act + row * s.nb_tok + block_offset(a, s, b);
            float x[32];
            if constexpr (VEC) {
                uint4 raw[TYPE == KVM_TYPE_F32 ? 8 : 4];
#pragma unroll
                for (int k = 0; k < (TYPE == KVM_TYPE_F32 ? 8 : 4); ++k) raw[k] = reinterpret_cast<const uint4 *>(src)[k];
                const uint8_t *p = reinterpret_cast<const uint8_t *>(raw);
#pragma unroll
                for (int e = 0; e < 32; ++e) x[e] = act_load<TYPE>(p + e * (TYPE == KVM_TYPE_F32 ? 4 : 2));
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) x[e] = act_load<TYPE>(src + e * s.nb_dim);
            }
            write_block<CT>(x, words ? mine + lane * bb : dst);
        }
        if (words) {
            __syncwarp();
            constexpr int per = bb / 2;                  // words of a pair
            const uint32_t ok = __ballot_sync(0xffffffffu, on);
            const uint64_t base = reinterpret_cast<uint64_t>(dst);
#pragma unroll
            for (int y = 0; y < (16 * per + 31) / 32; ++y) {
                const int w = lane + 32 * y, pair = min(w / per, 15), at = w - pair * per;
                uint8_t *to = reinterpret_cast<uint8_t *>(__shfl_sync(0xffffffffu, base, 2 * pair));
                if (w < 16 * per && ((ok >> (2 * pair)) & 1u))
                    reinterpret_cast<uint32_t *>(to)[at] = *reinterpret_cast<const uint32_t *>(mine + w * 4);
            }
            __syncwarp();
        }
    }
}

template <int TYPE, bool VEC>
__global__ void __launch_bounds__(kRowsThreads, 4) write_rows_kernel(const __grid_constant__ RowsArgs a) {
    __shared__ __align__(16) uint8_t stage[kRowsThreads * kBlockBytesQ8];
    const RowsSide &s = a.side[blockIdx.y];
    if (!s.on) return;
    if (s.cache_type == KVM_TYPE_Q4_0) write_side<TYPE, VEC, KVM_TYPE_Q4_0>(a, s, stage);
    else if (s.cache_type == KVM_TYPE_Q5_0) write_side<TYPE, VEC, KVM_TYPE_Q5_0>(a, s, stage);
    else if (s.cache_type == KVM_TYPE_Q8_0) write_side<TYPE, VEC, KVM_TYPE_Q8_0>(a, s, stage);
    else write_side<TYPE, VEC, KVM_TYPE_F16>(a, s, stage);
}

// A thread two runs of eight values, 8 c .. 8 c + 7 of a block and the same 16
// further on: in the 4- and 5-bit types the two share their bytes.
template <int TYPE, bool VEC, int CT>
__device__ __forceinline__ void read_side(const RowsArgs &a, const RowsSide &s) {
    constexpr int bb = block_bytes(CT);
    const uint64_t all = static_cast<uint64_t>(a.n) * a.blocks * 2u;
    auto u16 = [](const uint8_t *q) { return static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(q)); };
    for (uint64_t i = blockIdx.x * static_cast<uint64_t>(kRowsThreads) + threadIdx.x; i < all;
         i += static_cast<uint64_t>(gridDim.x) * kRowsThreads) {
        const uint32_t row = a.row(i), in_row = static_cast<uint32_t>(i - static_cast<uint64_t>(row) * (2u * a.blocks));
        const uint32_t b = in_row >> 1, c = in_row & 1u;
        const int64_t cell = a.cells[row];
        float x[16];
        if (cell < 0 || cell >= a.n_cells) {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = 0.0f;
        } else {
            const uint8_t *p = s.cache + static_cast<uint64_t>(cell) * s.row_bytes + static_cast<uint64_t>(b) * bb;
            if constexpr (CT == KVM_TYPE_F16) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    x[e] = __half2float(__ushort_as_half(static_cast<uint16_t>(u16(p + 16 * c + 2 * (e & 7) + 32 * (e >> 3)))));
            } else {
                const float d = __half2float(__ushort_as_half(static_cast<uint16_t>(u16(p))));
                if constexpr (CT == KVM_TYPE_Q8_0) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t w = u16(p + 2 + 8 * c + 2 * (e & 3) + 16 * (e >> 2));
                        x[2 * e] = d * static_cast<float>(static_cast<int8_t>(w & 255u));
                        x[2 * e + 1] = d * static_cast<float>(static_cast<int8_t>(w >> 8));
                    }
                } else {
                    constexpr bool q5 = CT == KVM_TYPE_Q5_0;
                    constexpr int mid = q5 ? 16 : 8;
                    // the fifth bits of values 8 c and on in bits 0-7, of those 16 further on in 16-23
                    const uint32_t fifth = q5 ? (u16(p + 2) | u16(p + 4) << 16) >> (8 * c) : 0u;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t w = u16(p + bb - 16 + 8 * c + 2 * e);
                        uint32_t q[4] = {w & 15u, (w >> 8) & 15u, (w >> 4) & 15u, w >> 12};
                        if (q5) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) q[k] |= ((fifth >> (2 * e + (k & 1) + 16 * (k >> 1))) & 1u) << 4;
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[2 * e + (k & 1) + 8 * (k >> 1)] = d * static_cast<float>(static_cast<int>(q[k]) - mid);
                    }
                }
            }
        }
        uint8_t *first = s.act + row * s.nb_tok + block_offset(a, s, b) + 8 * c * s.nb_dim;
#pragma unroll
        for (int k = 0; k < 16; k += 8) {
            uint8_t *dst = first + 2 * k * s.nb_dim;
            if constexpr (VEC && TYPE == KVM_TYPE_F32) {
                reinterpret_cast<float4 *>(dst)[0] = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
                reinterpret_cast<float4 *>(dst)[1] = make_float4(x[k + 4], x[k + 5], x[k + 6], x[k + 7]);
            } else if constexpr (VEC) {
                *reinterpret_cast<uint4 *>(dst) = make_uint4(act_pack<TYPE>(x[k], x[k + 1]), act_pack<TYPE>(x[k + 2], x[k + 3]),
                                                             act_pack<TYPE>(x[k + 4], x[k + 5]), act_pack<TYPE>(x[k + 6], x[k + 7]));
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) act_store<TYPE>(dst + e * s.nb_dim, x[k + e]);
            }
        }
    }
}

template <int TYPE, bool VEC>
__global__ void __launch_bounds__(kRowsThreads) read_rows_kernel(const __grid_constant__ RowsArgs a) {
    const RowsSide &s = a.side[blockIdx.y];
    if (!s.on) return;
    if (s.cache_type == KVM_TYPE_Q4_0) read_side<TYPE, VEC, KVM_TYPE_Q4_0>(a, s);
    else if (s.cache_type == KVM_TYPE_Q5_0) read_side<TYPE, VEC, KVM_TYPE_Q5_0>(a, s);
    else if (s.cache_type == KVM_TYPE_Q8_0) read_side<TYPE, VEC, KVM_TYPE_Q8_0>(a, s);
    else read_side<TYPE, VEC, KVM_TYPE_F16>(a, s);
}

kvm_status rows_call(const char *me, bool write, kvm_stream stream, const kvm_cache *c, uint32_t n,
                     const int64_t *d_cells, const kvm_rows *k, const kvm_rows *v) {
    kvm_status r = cache_check(c, me);
    if (r != KVM_OK) return r;
    if (!k && !v) return layer_fail(KVM_EINVAL, "%s: neither k nor v", me);
    if (n > 0x7fffffffu) return layer_fail(KVM_EINVAL, "%s: too many rows", me);
    if (n == 0) return KVM_OK;
    if (k && (r = rows_check(k, c->n_head_kv, c->head_dim, me)) != KVM_OK) return r;
    if (v && (r = rows_check(v, c->n_head_kv, c->head_dim, me)) != KVM_OK) return r;
    if (k && v && k->type != v->type) return layer_fail(KVM_EINVAL, "%s: k and v must have one type", me);
    if (!d_cells || (reinterpret_cast<uintptr_t>(d_cells) & 7u))
        return layer_fail(KVM_EINVAL, "%s: cells must be an 8-byte aligned array", me);
    PointerDevice dev(c->d_k, me);
    if (dev.status() != KVM_OK) return dev.status();
    RowsArgs a{};
    const uint32_t width = c->n_head_kv * c->head_dim;
    a.cells = d_cells;
    a.n_cells = static_cast<int64_t>(c->block_tokens) * c->n_slots;
    a.n = n;
    a.blocks = width / 32u;
    a.head_blocks = c->head_dim / 32u;
    a.row = Divide::by(a.blocks * (write ? 1u : 2u));
    a.head = Divide::by(a.head_blocks);
    for (int i = 0; i < 2; ++i) {
        const kvm_rows *x = i ? v : k;
        RowsSide &s = a.side[i];
        s.on = x != nullptr;
        if (!x) continue;
        s.cache = static_cast<uint8_t *>(i ? c->d_v : c->d_k);
        s.cache_type = i ? c->type_v : c->type_k;
        s.row_bytes = kvm_row_bytes(s.cache_type, width);
        s.act = static_cast<uint8_t *>(const_cast<void *>(x->data));
        s.nb_dim = x->nb_dim;
        s.nb_head = x->nb_head;
        s.nb_tok = x->nb_tok;
    }
    const uint64_t want = (static_cast<uint64_t>(n) * a.blocks * (write ? 1u : 2u) + kRowsThreads - 1) / kRowsThreads;
    const uint64_t most = 32ull * num_sms();
    const dim3 grid(static_cast<uint32_t>(want < most ? want : most), 2);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int32_t type = (k ? k : v)->type;
    const bool vec = (!k || rows_vec16(k)) && (!v || rows_vec16(v));
    auto go = [&](auto ty) {
        constexpr int T = decltype(ty)::value;
        if (write && vec) write_rows_kernel<T, true><<<grid, kRowsThreads, 0, st>>>(a);
        else if (write) write_rows_kernel<T, false><<<grid, kRowsThreads, 0, st>>>(a);
        else if (vec) read_rows_kernel<T, true><<<grid, kRowsThreads, 0, st>>>(a);
        else read_rows_kernel<T, false><<<grid, kRowsThreads, 0, st>>>(a);
    };
    if (type == KVM_TYPE_F32) go(std::integral_constant<int, KVM_TYPE_F32>{});
    else if (type == KVM_TYPE_F16) go(std::integral_constant<int, KVM_TYPE_F16>{});
    else go(std::integral_constant<int, KVM_TYPE_BF16>{});
    return layer_cuda(cudaGetLastError(), me);
}

}  // namespace
}  // namespace kvm

using namespace kvm;

extern "C" kvm_status kvm_write_rows(kvm_stream stream, const kvm_cache *cache, uint32_t n, const int64_t *d_cells,
                                     const kvm_rows *k, const kvm_rows *v) {
    return rows_call("kvm_write_rows", true, stream, cache, n, d_cells, k, v);
}

extern "C" kvm_status kvm_read_rows(kvm_stream stream, const kvm_cache *cache, uint32_t n, const int64_t *d_cells,
                                    const kvm_rows *k_out, const kvm_rows *v_out) {
    return rows_call("kvm_read_rows", false, stream, cache, n, d_cells, k_out, v_out);
}
