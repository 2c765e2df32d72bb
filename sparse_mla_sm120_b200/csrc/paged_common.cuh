// What the kernels of attention over a block table share (paged.cu, paged_pair.cu): how requests' rows are cut into partitions, masks of
// the LSE, 16-bit forms.
#pragma once

#include "attn_common.cuh"
#include "sm100_ptx.cuh"

namespace smla {

namespace {

using namespace ptx;
using namespace attn;

// Blocks' worth of time that a request takes before its first row; no partition is shorter.  (Partitions of four blocks at least, for less
// to merge where SMs are idle: one request of 1000 rows, 16 heads, 15.2 us instead of 13.3.)
constexpr int PG_START = 2;
// The running maximum of a row lags by at most 2^PG_TAU: weights are floating point, so that costs no precision (fp16 weights reach
// 2^8 and fall to zero 2^-24 below a maximum that does not lag), and the accumulator is rescaled a few times per request.
constexpr float PG_TAU = 8.0f;
constexpr float NO_RECORD = -INFINITY;            // the LSE of a partition's record in which a query row sees nothing (scores may lie below NEG_BIG)
constexpr uint32_t G_CHUNK = 64 * 128;            // 64 dims of 64 rows, 128B swizzle

__device__ __forceinline__ uint32_t gswz(uint32_t row, uint32_t piece) { return row * 128u + ((piece ^ (row & 7u)) << 4); }

__device__ __forceinline__ int paged_length(const PagedParams& p, int req) {
    const long long most = (long long)p.pages_per_request * p.page_block_size;
    const int n = max(ld_in(p.lengths + req), 0);
    return n < most ? n : (int)most;
}
template <int ROWS> __device__ __forceinline__ int paged_blocks(int len) { return (int)(((unsigned)len + (ROWS - 1u)) / (unsigned)ROWS); }
__device__ __forceinline__ long long paged_share(long long total, int parts) {
    // (a 64-bit division takes hundreds of cycles)
    const long long u = total + parts <= 0xffffffffll ? (long long)((unsigned)(total + parts - 1) / (unsigned)parts) : (total + parts - 1) / parts;
    return u > PG_START ? u : PG_START;
}

// The pieces of a partition, one after the other: request, its rows, and which of its blocks of ROWS rows are the partition's.
template <int ROWS> struct Pieces {
    long long lo, hi;                     // the partition's part of the line, from where the request begins on it
    int req, len, nb, b0, b1;
    __device__ __forceinline__ bool next(const PagedParams& p) {
        while (true) {
            if (nb >= 0) { lo -= nb + PG_START; hi -= nb + PG_START; ++req; }
            if (req >= p.batch || hi <= 0) return false;
            len = paged_length(p, req);
            nb = paged_blocks<ROWS>(len);
            b0 = (int)max(lo - PG_START, 0ll);
            b1 = (int)min(hi - PG_START, (long long)nb);
            if (b1 > b0) return true;
            if (nb == 0 && PG_START - 1 >= lo && PG_START - 1 < hi) { b0 = b1 = 0; return true; }      // a request without rows: whoever holds its last unit
        }
    }
    __device__ __forceinline__ bool whole() const { return b0 == 0 && b1 == nb; }
    // What the merge needs to know, written by the partition that has the request's first block: the request's last partition.
    __device__ __forceinline__ void write_span(const PagedParams& p, int part, long long share) const {
        const long long more = nb + PG_START - hi;        // units behind this partition
        int last = part;
        if (!whole() && more > 0) last += more + share <= 0xffffffffll ? (int)((unsigned)(more + share - 1) / (unsigned)share) : (int)((more + share - 1) / share);
        p.spans[req] = make_int2(part, last);
    }
};

// How many partitions a request lies in, by its span; 0 where the words are none.  (A partition whose wait gave up has written no spans: the
// merge then finds what the scratch held before, and must not read outside of the records.)
__host__ __device__ inline int span_parts(int first, int last, int num_parts) { return first >= 0 && first <= last && last < num_parts ? last - first + 1 : 0; }

// The partition's part of the line: every thread sums the requests of its share, the block (of `warps` warps) scans the sums.  scan: 23
// words of shared memory; word 20 has the length of a part afterwards.  Synchronises the block, tensor memory's address included.
template <int ROWS> __device__ __forceinline__ Pieces<ROWS> partition_of(const PagedParams& p, int part, long long* scan, int warps) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int per = (p.batch + (int)blockDim.x - 1) / (int)blockDim.x;
    const int r_lo = min(tid * per, p.batch), r_hi = min(r_lo + per, p.batch);
    long long sum = 0;
    for (int r = r_lo; r < r_hi; ++r) sum += paged_blocks<ROWS>(paged_length(p, r)) + PG_START;
    long long incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    long long before = incl - sum, total = 0;
#pragma unroll
    for (int w = 0; w < warps; ++w) {
        if (w < warp) before += scan[w];
        total += scan[w];
    }
    const long long share = paged_share(total, p.num_parts), lo = min(part * share, total), hi = min(lo + share, total);
    if (before <= lo && lo < before + sum) {
        int r = r_lo;
        for (; r < r_hi - 1; ++r) {
            const int w = paged_blocks<ROWS>(paged_length(p, r)) + PG_START;
            if (lo < before + w) break;
            before += w;
        }
        scan[21] = before;
        scan[22] = r;
    }
    if (tid == 0) scan[20] = share;
    __syncthreads();
    Pieces<ROWS> piece;
    piece.req = lo < hi ? (int)scan[22] : p.batch;
    piece.lo = lo - scan[21];
    piece.hi = hi - scan[21];
    piece.nb = -1;                        // before the first
    return piece;
}

// Rows of the request that a query row sees: all, or up to the query's own.
__device__ __forceinline__ int paged_sees(const PagedParams& p, int len, int row) {
    if (!p.causal) return len;
    return min(max(len - (p.query_len - 1) + min(row, p.rows - 1) / p.num_heads, 0), len);
}

// log2(2^a + 2^b)
__device__ __forceinline__ float log2_add(float a, float b) {
    const float hi = fmaxf(a, b), lo = fminf(a, b);
    return (hi == INFINITY || hi == -INFINITY) ? hi : hi + log2f(1.f + exp2f(lo - hi));
}
// LSE of a row with a sink: `lse` is NEG_BIG where the row sees nothing.
__device__ __forceinline__ float with_sink(float lse, float sink2) {
    if (lse != NEG_BIG) return log2_add(lse, sink2);
    return sink2 == -INFINITY ? NEG_BIG : sink2;
}

template <bool F16> __device__ __forceinline__ uint32_t pack_weights(float a, float b) {
    if (F16) {
        const __half2 r = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <bool F16> __device__ __forceinline__ uint16_t out_bits(float v) {
    if (F16) return __half_as_ushort(__float2half_rn(v));
    return __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

// Values that are no numbers, replaced by zeros.
template <bool F16> __device__ __forceinline__ uint32_t numbers_only(uint32_t x) {
    constexpr uint32_t E = F16 ? 0x7c00u : 0x7f80u;
    if ((x & E) == E) x &= 0xffff0000u;
    if ((x & (E << 16)) == (E << 16)) x &= 0x0000ffffu;
    return x;
}
template <bool F16> __device__ __forceinline__ uint4 numbers_only(uint4 v) {
    return make_uint4(numbers_only<F16>(v.x), numbers_only<F16>(v.y), numbers_only<F16>(v.z), numbers_only<F16>(v.w));
}

}  // namespace

}  // namespace smla
