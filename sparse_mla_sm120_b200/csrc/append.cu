// What new tokens leave in the caches: latent rows (append_kv_kernel) and the indexer's keys (append_index_kernel), with the
// position rotation applied on the way, and the same tokens' queries.
//
// A pair (a, b) of the 64 rotated values turns by its token's angle: a' = a cos - b sin, b' = b cos + a sin, in fp32, rounded once to
// the type it is kept in.  Pairs are neighbours (2 i, 2 i + 1) or, for the other convention, i and i + 32; the angles' cosines and sines are
// the caller's table, fp32, 32 + 32 per position.
//
// Both kernels stream: a warp takes one token's row or a group of its heads' queries, all of its loads are asked for before the
// first is used, and nothing is read or written twice.  append_kv_kernel is bound by memory: 8192 tokens of 128 heads into 656-byte rows 53.9 us,
// 5.3 TB/s; 2047 of 64 heads, 584-byte rows 7.4 us, 5.0 TB/s; a single token 3.9 us, two waits for memory.
#include "common.cuh"

#include <type_traits>

namespace smla {

namespace {

constexpr int WARPS = 8;
constexpr int KV_HEADS = 16;      // heads of queries per warp of append_kv_kernel: four loads of 16 bytes per lane
constexpr int IX_HEADS = 8;       // of append_index_kernel

__device__ __forceinline__ float pow2_ceil(float x) {   // smallest power of two >= x (x > 0, normal)
    uint32_t b = __float_as_uint(x);
    if (b & 0x007fffffu) b = (b + 0x00800000u) & 0x7f800000u;
    return __uint_as_float(b);
}

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
}

// Slots and positions come as int32 or int64.
__device__ __forceinline__ int64_t ld_index(const void* p, int wide, int64_t i) {
    if (!wide) return ld_in(static_cast<const int*>(p) + i);
    const uint2 v = ld_in(static_cast<const uint2*>(p) + i);
    return (int64_t)(((uint64_t)v.y << 32) | v.x);
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {     // (values that are no number stay none)
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) |
           ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16);
}

// a / b of numbers that are not negative, in 32 bits where they suffice (a 64-bit division takes a warp a hundred instructions).
__device__ __forceinline__ int64_t quotient(int64_t a, int b) { return a <= 0xffffffffll ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b; }

// The 64 values of a rotated vector by eight lanes, eight values each: [8 l, 8 l + 8) where pairs are neighbours, else [4 l, 4 l + 4)
// and the same 32 further.
template <bool PAIRS> __device__ __forceinline__ uint4 ld_rot(const uint16_t* p, int l) {
    if (PAIRS) return ld_in_once(reinterpret_cast<const uint4*>(p + 8 * l));
    const uint2 a = ld_in_once(reinterpret_cast<const uint2*>(p + 4 * l)), b = ld_in_once(reinterpret_cast<const uint2*>(p + 32 + 4 * l));
    return make_uint4(a.x, a.y, b.x, b.y);
}
template <bool PAIRS> __device__ __forceinline__ void st_rot(uint16_t* p, int l, uint4 v) {
    if (PAIRS) {
        *reinterpret_cast<uint4*>(p + 8 * l) = v;
    } else {
        *reinterpret_cast<uint2*>(p + 4 * l) = make_uint2(v.x, v.y);
        *reinterpret_cast<uint2*>(p + 32 + 4 * l) = make_uint2(v.z, v.w);
    }
}
// c and s: cosines and sines of angles [4 l, 4 l + 4).
template <typename T, bool PAIRS> __device__ __forceinline__ uint4 rotate(uint4 v, float4 c, float4 s) {
    const float2 x0 = unpack2<T>(v.x), x1 = unpack2<T>(v.y), x2 = unpack2<T>(v.z), x3 = unpack2<T>(v.w);
    if (PAIRS)
        return make_uint4(pack2<T>(x0.x * c.x - x0.y * s.x, x0.y * c.x + x0.x * s.x), pack2<T>(x1.x * c.y - x1.y * s.y, x1.y * c.y + x1.x * s.y),
                          pack2<T>(x2.x * c.z - x2.y * s.z, x2.y * c.z + x2.x * s.z), pack2<T>(x3.x * c.w - x3.y * s.w, x3.y * c.w + x3.x * s.w));
    return make_uint4(pack2<T>(x0.x * c.x - x2.x * s.x, x0.y * c.y - x2.y * s.y), pack2<T>(x1.x * c.z - x3.x * s.z, x1.y * c.w - x3.y * s.w),
                      pack2<T>(x2.x * c.x + x0.x * s.x, x2.y * c.y + x0.y * s.y), pack2<T>(x3.x * c.z + x1.x * s.z, x3.y * c.w + x1.y * s.w));
}

// One warp: the row of a token (part 0 of its 1 + ceil(heads / 16)), or the queries of 16 of its heads.
template <int LAYOUT, bool PAIRS> __global__ void __launch_bounds__(WARPS * 32) append_kv_kernel(const AppendKvParams p) {
    typedef typename std::conditional<LAYOUT == SMLA_LAYOUT_F16, __half, __nv_bfloat16>::type T;
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
    const int64_t t = quotient(unit, p.parts);
    const int part = (int)(unit - t * p.parts), l = lane & 7;
    if (t >= p.num_tokens) return;
    float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
    // The values are asked for before the position, the table's entry and the slot are known: else a warp waits for memory two or three
    // times in a row (8192 tokens of 128 heads 64.1 -> 53.9 us).
    const int64_t pos = p.positions != nullptr ? ld_index(p.positions, p.positions64, t) : 0;
    const bool lost = p.positions != nullptr && (pos < 0 || pos >= p.num_positions);       // a token without a position leaves nothing, or zeros in q_out
    if (part > 0) {
        const uint16_t* src = p.q_pe + t * p.q_pe_token;
        uint16_t* dst = p.q_out + t * p.q_out_token;
        const int h0 = (part - 1) * KV_HEADS + (lane >> 3);
        uint4 v[KV_HEADS / 4];
#pragma unroll
        for (int i = 0; i < KV_HEADS / 4; ++i)
            if (h0 + 4 * i < p.num_heads) v[i] = ld_rot<PAIRS>(src + (h0 + 4 * i) * p.q_pe_head, l);
        if (lost) {
            if (p.clear_lost) {
#pragma unroll
                for (int i = 0; i < KV_HEADS / 4; ++i)
                    if (h0 + 4 * i < p.num_heads) st_rot<PAIRS>(dst + (h0 + 4 * i) * p.q_out_head, l, make_uint4(0, 0, 0, 0));
            }
            return;
        }
        c = ld_in(reinterpret_cast<const float4*>(p.cos_sin + pos * 64) + l);
        s = ld_in(reinterpret_cast<const float4*>(p.cos_sin + pos * 64 + 32) + l);
#pragma unroll
        for (int i = 0; i < KV_HEADS / 4; ++i)
            if (h0 + 4 * i < p.num_heads) st_rot<PAIRS>(dst + (h0 + 4 * i) * p.q_out_head, l, rotate<T, PAIRS>(v[i], c, s));
        return;
    }
    const int64_t slot = ld_index(p.slots, p.slots64, t);
    const uint16_t* src = p.kv_c + t * p.kv_c_token;
    constexpr int NOPE = LAYOUT == SMLA_LAYOUT_MODEL1 ? 448 : 512;
    const bool mine = LAYOUT != SMLA_LAYOUT_MODEL1 || lane < 28;
    // 16-bit rows are copied, a lane's two pieces 512 bytes apart; packed rows: a lane takes 16 neighbours
    constexpr bool ROWS16 = LAYOUT == SMLA_LAYOUT_BF16 || LAYOUT == SMLA_LAYOUT_F16;
    uint4 a = make_uint4(0, 0, 0, 0), b = a, r = a;
    if (mine) {
        a = ld_in_once(reinterpret_cast<const uint4*>(src + lane * (ROWS16 ? 8 : 16)));
        b = ld_in_once(reinterpret_cast<const uint4*>(src + (ROWS16 ? 256 + lane * 8 : lane * 16 + 8)));
    }
    if (lane < 8) r = ld_rot<PAIRS>(p.k_pe + t * p.k_pe_token, l);
    if (lost || slot < 0 || slot >= p.capacity) return;
    const int64_t page = quotient(slot, p.page_block_size);
    const int in = (int)(slot - page * p.page_block_size);
    uint8_t* base = p.cache + page * p.page_stride;
    if (lane < 8) {
        if (p.positions != nullptr) {
            c = ld_in(reinterpret_cast<const float4*>(p.cos_sin + pos * 64) + l);
            s = ld_in(reinterpret_cast<const float4*>(p.cos_sin + pos * 64 + 32) + l);
            r = rotate<T, PAIRS>(r, c, s);
        }
    }
    if (ROWS16) {
        uint16_t* dst = reinterpret_cast<uint16_t*>(base + (int64_t)in * (2 * D_QK));
        *reinterpret_cast<uint4*>(dst + lane * 8) = a;
        *reinterpret_cast<uint4*>(dst + 256 + lane * 8) = b;
        if (lane < 8) st_rot<PAIRS>(dst + NOPE, l, r);
        return;
    }
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    float v[16];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 x = unpack2<__nv_bfloat16>(w[i]);
        v[2 * i] = x.x; v[2 * i + 1] = x.y;
        amax = fmaxf(amax, fmaxf(fabsf(x.x), fabsf(x.y)));
    }
    // a scale stands for 128 values (8 lanes), or 64 (4)
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    if (LAYOUT == SMLA_LAYOUT_V32) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 4));
    const float scale = pow2_ceil(fmaxf(fmaxf(amax, 1e-4f) / 448.f, 1e-4f));
    const float inv = 1.f / scale;  // exact: power of two
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = e4m3x4(v[4 * i] * inv, v[4 * i + 1] * inv, v[4 * i + 2] * inv, v[4 * i + 3] * inv);
    if (LAYOUT == SMLA_LAYOUT_V32) {
        uint8_t* dst = base + (int64_t)in * ROW_BYTES;
        *reinterpret_cast<uint4*>(dst + lane * 16) = make_uint4(o[0], o[1], o[2], o[3]);
        if ((lane & 7) == 0) *reinterpret_cast<float*>(dst + SCALE_OFF + (lane >> 3) * 4) = scale;
        if (lane < 8) st_rot<PAIRS>(reinterpret_cast<uint16_t*>(dst + ROPE_OFF), l, r);
    } else {
        // pages of an odd number of rows start on 8 bytes only
        uint8_t* dst = base + (int64_t)in * SMLA_M1_DATA_BYTES;
        if (mine) {
            *reinterpret_cast<uint2*>(dst + lane * 16) = make_uint2(o[0], o[1]);
            *reinterpret_cast<uint2*>(dst + lane * 16 + 8) = make_uint2(o[2], o[3]);
        }
        uint32_t e = 0u;                                       // lane i: exponent i of the footer, 0 in the eighth
        e = __shfl_sync(0xffffffffu, __float_as_uint(scale) >> 23, (lane & 7) * 4);
        if ((lane & 7) == 7) e = 0u;
        uint32_t lo = 0u, hi = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lo |= __shfl_sync(0xffffffffu, e, i) << (8 * i);
            hi |= __shfl_sync(0xffffffffu, e, 4 + i) << (8 * i);
        }
        if (lane == 0) *reinterpret_cast<uint2*>(base + (int64_t)p.page_block_size * SMLA_M1_DATA_BYTES + (int64_t)in * 8) = make_uint2(lo, hi);
        if (lane < 8) {
            uint16_t* rope = reinterpret_cast<uint16_t*>(dst + NOPE);
            if (PAIRS) {
                *reinterpret_cast<uint2*>(rope + 8 * l) = make_uint2(r.x, r.y);
                *reinterpret_cast<uint2*>(rope + 8 * l + 4) = make_uint2(r.z, r.w);
            } else {
                st_rot<false>(rope, l, r);
            }
        }
    }
}

// One warp: a token's key (part 0), or the queries of eight of its heads; 16 lanes per row, eight values each.
// x -> rotated in fp32, scale = max(|x|, 1e-4) / 448 over the row, e4m3(x / scale).  A query's scale goes into its head's weight.
// What bounds it is the issue of instructions, 227 for 256 values (65 % of the slots): 4096 tokens of 64 heads 40.4 us, 2.6 TB/s.  Measured and not
// kept: eight lanes per row, so that all lanes turn values (half the instructions, but 71 registers: 46.3; 64 with spills: 40.6).
template <bool PAIRS> __global__ void __launch_bounds__(WARPS * 32) append_index_kernel(const AppendIndexParams p) {
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, l = lane & 15;
    const int64_t unit = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
    const int64_t t = quotient(unit, p.parts);
    const int part = (int)(unit - t * p.parts);
    if (t >= p.num_tokens) return;
    const int64_t pos = p.positions != nullptr ? ld_index(p.positions, p.positions64, t) : 0;
    constexpr int N = IX_HEADS / 2;
    const int rows = part == 0 ? 1 : min(p.num_heads - (part - 1) * IX_HEADS, IX_HEADS);
    const int64_t row0 = part == 0 ? t : t * p.num_heads + (part - 1) * IX_HEADS;
    const uint16_t* src = part == 0 ? p.k + t * p.k_token : p.q + row0 * 128;
    uint4 v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = make_uint4(0, 0, 0, 0);
        if (2 * i + (lane >> 4) < rows) v[i] = ld_in_once(reinterpret_cast<const uint4*>(src + (2 * i + (lane >> 4)) * 128 + l * 8));
    }
    int64_t slot = 0;
    if (part == 0) slot = ld_index(p.slots, p.slots64, t);
    if (p.positions != nullptr && (pos < 0 || pos >= p.num_positions)) {        // no key; queries of zeros and weight zero
        if (part > 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = 2 * i + (lane >> 4);
                if (r >= rows) break;
                *reinterpret_cast<uint2*>(p.qi + (row0 + r) * 128 + l * 8) = make_uint2(0, 0);
                if (l == 0) p.w_out[row0 + r] = 0.f;
            }
        }
        return;
    }
    // the rotated half of the row lies in eight neighbouring lanes
    const bool turns = p.positions != nullptr && (l >> 3) == (p.rope_offset >> 6);
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { c[i] = 1.f; s[i] = 0.f; }
    if (turns) {
        const float* cs = p.cos_sin + pos * 64;
        if (PAIRS) {
            const float4 a = ld_in(reinterpret_cast<const float4*>(cs) + (l & 7)), b = ld_in(reinterpret_cast<const float4*>(cs + 32) + (l & 7));
            c[0] = a.x; c[1] = a.y; c[2] = a.z; c[3] = a.w;
            s[0] = b.x; s[1] = b.y; s[2] = b.z; s[3] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float4 a = ld_in(reinterpret_cast<const float4*>(cs) + 2 * (l & 3) + i), b = ld_in(reinterpret_cast<const float4*>(cs + 32) + 2 * (l & 3) + i);
                c[4 * i] = a.x; c[4 * i + 1] = a.y; c[4 * i + 2] = a.z; c[4 * i + 3] = a.w;
                s[4 * i] = b.x; s[4 * i + 1] = b.y; s[4 * i + 2] = b.z; s[4 * i + 3] = b.w;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (2 * i >= rows) break;
        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 y = unpack2<__nv_bfloat16>(w[j]);
            x[2 * j] = y.x; x[2 * j + 1] = y.y;
        }
        if (PAIRS) {
            if (turns) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float a = x[2 * j], b = x[2 * j + 1];
                    x[2 * j] = a * c[j] - b * s[j];
                    x[2 * j + 1] = b * c[j] + a * s[j];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {                     // the other of the pair lies four lanes away
                const float y = __shfl_xor_sync(0xffffffffu, x[j], 4);
                if (turns) x[j] = x[j] * c[j] + ((l & 4) ? y : -y) * s[j];
            }
        }
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[j]));
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const float scale = __fdiv_rn(fmaxf(amax, 1e-4f), 448.f), inv = __fdiv_rn(1.f, scale);
        // x / scale, rounded to fp32 and then to e4m3.  x inv lies within two steps of fp32 of it, so both give the same e4m3 value unless a
        // border of e4m3's rounding (the middle of two of its values: 20 bits of the fp32 mantissa say 1000...) is as near; only then,
        // once in some 30000 values, and below e4m3's normal range, the warp divides.  (A division takes some ten instructions.)
        float z[8];
        bool near = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            z[j] = x[j] * inv;
            near |= ((__float_as_uint(z[j]) - 0x7fffdu) & 0xfffffu) <= 6u || fabsf(z[j]) < 0x1p-6f;
        }
        if (near) {
#pragma unroll
            for (int j = 0; j < 8; ++j) z[j] = __fdiv_rn(x[j], scale);
        }
        const uint2 y = make_uint2(e4m3x4(z[0], z[1], z[2], z[3]), e4m3x4(z[4], z[5], z[6], z[7]));
        const int r = 2 * i + (lane >> 4);
        if (r >= rows) continue;
        if (part == 0) {
            if (slot < 0 || slot >= p.capacity) continue;
            *reinterpret_cast<uint2*>(p.ki + slot * 128 + l * 8) = y;
            if (l == 0) p.k_scale[slot] = scale;
        } else {
            *reinterpret_cast<uint2*>(p.qi + (row0 + r) * 128 + l * 8) = y;
            if (l == 0) p.w_out[row0 + r] = p.weights != nullptr ? ld_in(p.weights + row0 + r) * scale : scale;
        }
    }
}

}  // namespace

int launch_append_kv(AppendKvParams p, int layout, bool pairs, cudaStream_t stream) {
    if (p.num_tokens == 0) return 0;
    p.parts = 1 + (p.q_pe != nullptr ? (p.num_heads + KV_HEADS - 1) / KV_HEADS : 0);
    const int64_t blocks = ((int64_t)p.num_tokens * p.parts + WARPS - 1) / WARPS;
    if (blocks > 0x7fffffff) return set_error(SMLA_E_SHAPE, "append_kv_kernel: %d tokens of %d heads", p.num_tokens, p.num_heads);
    typedef void (*Kernel)(const AppendKvParams);
    Kernel kernel;
    switch (layout) {
        case SMLA_LAYOUT_V32: kernel = pairs ? append_kv_kernel<SMLA_LAYOUT_V32, true> : append_kv_kernel<SMLA_LAYOUT_V32, false>; break;
        case SMLA_LAYOUT_MODEL1: kernel = pairs ? append_kv_kernel<SMLA_LAYOUT_MODEL1, true> : append_kv_kernel<SMLA_LAYOUT_MODEL1, false>; break;
        case SMLA_LAYOUT_BF16: kernel = pairs ? append_kv_kernel<SMLA_LAYOUT_BF16, true> : append_kv_kernel<SMLA_LAYOUT_BF16, false>; break;
        default: kernel = pairs ? append_kv_kernel<SMLA_LAYOUT_F16, true> : append_kv_kernel<SMLA_LAYOUT_F16, false>; break;
    }
    launch_dependent(kernel, dim3((unsigned)blocks), dim3(WARPS * 32), 0, stream, p);
    return check_launch("append_kv_kernel");
}

int launch_append_index(AppendIndexParams p, bool pairs, cudaStream_t stream) {
    if (p.num_tokens == 0) return 0;
    p.parts = 1 + (p.q != nullptr ? (p.num_heads + IX_HEADS - 1) / IX_HEADS : 0);
    const int64_t blocks = ((int64_t)p.num_tokens * p.parts + WARPS - 1) / WARPS;
    if (blocks > 0x7fffffff) return set_error(SMLA_E_SHAPE, "append_index_kernel: %d tokens of %d heads", p.num_tokens, p.num_heads);
    launch_dependent(pairs ? append_index_kernel<true> : append_index_kernel<false>, dim3((unsigned)blocks), dim3(WARPS * 32), 0, stream, p);
    return check_launch("append_index_kernel");
}

}  // namespace smla
