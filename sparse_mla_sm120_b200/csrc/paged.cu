// Attention of a request's newest tokens over all of its rows, found through a block table (attn_paged_kernel), and the merge of what
// the partitions of a request leave (paged_combine_kernel).
//
//   s_j = scale q . k_j,  m = max_j s_j,  out = sum_j e^(s_j - m) v_j / (sum_j e^(s_j - m) + e^(sink - m)),  one pass over the rows with
// the running maximum and sum; nothing below the cache's 16-bit values and fp32 sums is rounded but the weights' 16-bit form for P.V.
//
// Work: all rows of all requests lie in one line of 64-row blocks, every request behind PG_START blocks' worth of nothing (what a
// request costs before its first row), and partition c takes the c-th equal piece of the line.  A request within one partition is
// written out directly; of others every partition leaves a normalised fp32 record with its LSE, and the merge joins them in order:
// results do not depend on timing.  The partitions find their pieces themselves, from the lengths: no scheduler launch.
//
// A CTA serves 64 query rows (heads of the newest tokens, token-major) of a partition:
//   S [64 x 64] = Q . K^T: A = Q, B = 64 cache rows, both K-major in chunks of 64 dims, 128B swizzle;
//   O^T [4 x 128 dims x rows] += V^T . P^T: A = the same rows read MN-major, B = the weights, a line of 64 rows' weights per query row.
// O has to be transposed: 64 x 512 fp32 fill half of tensor memory that way, all of it the other way.
// Warps: 0-3 softmax, epilogue; 4-7 and 8-11 bring the rows of even and odd blocks into two stages of 72 KB, 16-bit rows by
// cp.async, packed rows through registers (e4m3 x its scale is exact in bf16); 12 issues the MMAs: scores of a block as soon as its
// rows are there, P.V of the one before as soon as its weights are.
// Every wait is bounded; a wait that gives up records a code in status[] and the CTA drains and exits.
#include "attn_common.cuh"
#include "sm100_ptx.cuh"

namespace smla {

namespace {

using namespace ptx;
using namespace attn;

constexpr int PG_ROWS = 64;                       // query rows of a CTA
constexpr int PG_START = 2;                       // blocks' worth of time that a request takes before its first row
constexpr int PG_LEAST = 2;                       // blocks of rows that a partition should be worth
constexpr int PG_SM_WARPS = 4, PG_LD_WARPS = 8, PG_MMA_WARP = PG_SM_WARPS + PG_LD_WARPS;
constexpr int PG_THREADS = (PG_MMA_WARP + 1) * 32;
// The running maximum of a row lags by at most 2^PG_TAU: weights are floating point, so that costs no precision (fp16 weights reach
// 2^8 and fall to zero 2^-24 below a maximum that does not lag), and the accumulator is rescaled a few times per request.
constexpr float PG_TAU = 8.0f;

constexpr uint32_t G_CHUNK = 64 * 128;            // 64 dims of 64 rows
constexpr uint32_t G_STAGE = 9 * G_CHUNK;
constexpr uint32_t GQ_OFF = 0;
constexpr uint32_t GK_OFF = GQ_OFF + G_STAGE;
constexpr uint32_t GP_OFF = GK_OFF + 2 * G_STAGE;             // weights [64 query rows][64 rows] 16-bit
constexpr uint32_t GV_OFF = GP_OFF + G_CHUNK;                 // validity: a bit per row, [2 stages] 64 bits
constexpr uint32_t GN_OFF = GV_OFF + 16;                      // rows that some query must not see and whose values are no numbers
constexpr uint32_t GA_OFF = GN_OFF + 16;                      // [64] fp32: rescale factors, then 1 / denominator
constexpr uint32_t GW_OFF = GA_OFF + PG_ROWS * 4;             // schedule: block scan [16] int64, start int64, request, total
constexpr uint32_t GB_OFF = GW_OFF + 16 * 8 + 32;
constexpr int GB_KFULL = 0, GB_KFREE = 2, GB_SREADY = 4, GB_PREADY = 6, GB_PVDONE = 7, GB_QFREE = 8, GB_N = 9;
constexpr uint32_t GMISC_OFF = GB_OFF + GB_N * 8;
constexpr uint32_t G_SMEM = GMISC_OFF + 16 + 1024;
static_assert(G_SMEM <= 227 * 1024, "shared memory budget");
static_assert(GB_OFF % 8 == 0 && GA_OFF % 16 == 0 && GW_OFF % 8 == 0, "alignment");

constexpr uint32_t GT_O = 0, GT_S = 256;          // tensor memory: dims block b of O^T at 64 b, the two score buffers at 256 and 320
constexpr uint32_t G_DESC_HI = desc_hi(1024, (uint32_t)SWIZZLE_128B);

enum { WP_KFULL = 61, WP_KFREE = 62, WP_SREADY = 63, WP_PREADY = 64, WP_PVDONE = 65, WP_QFREE = 66 };

__device__ __forceinline__ uint32_t gswz(uint32_t row, uint32_t piece) { return row * 128u + ((piece ^ (row & 7u)) << 4); }

__device__ __forceinline__ int paged_length(const PagedParams& p, int req) {
    const long long most = (long long)p.pages_per_request * p.page_block_size;
    const int n = max(ld_in(p.lengths + req), 0);
    return n < most ? n : (int)most;
}
__device__ __forceinline__ int paged_blocks(int len) { return (int)(((unsigned)len + 63u) >> 6); }
__host__ __device__ __forceinline__ long long paged_share(long long total, int parts) {
    const long long u = (total + parts - 1) / parts;
    return u > PG_START + PG_LEAST ? u : PG_START + PG_LEAST;
}

// The pieces of a partition, one after the other: request, its rows, and which of its blocks are the partition's.
struct Pieces {
    long long lo, hi, start;       // the partition's part of the line, and where the request begins on it
    int req, len, nb, b0, b1;
    bool begun;
    __device__ __forceinline__ Pieces(long long lo_, long long hi_, int req_, long long start_) : lo(lo_), hi(hi_), start(start_), req(req_), begun(false) {}
    __device__ __forceinline__ bool next(const PagedParams& p) {
        while (true) {
            if (begun) { start += nb + PG_START; ++req; }
            begun = true;
            if (req >= p.batch || start >= hi) return false;
            len = paged_length(p, req);
            nb = paged_blocks(len);
            const long long first = start + PG_START;
            b0 = (int)max(lo - first, 0ll);
            b1 = (int)min(hi - first, (long long)nb);
            if (b1 > b0) return true;
            if (nb == 0 && first - 1 >= lo && first - 1 < hi) { b0 = b1 = 0; return true; }      // a request without rows: whoever holds its last unit
        }
    }
    __device__ __forceinline__ bool whole() const { return b0 == 0 && b1 == nb; }
};

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

// Sixteen e4m3 values times their scale as bf16 (exact for powers of two; no number stays none).
__device__ __forceinline__ void dequant16(uint4 v, float scale, uint32_t (&d)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i] >> (16 * h)), __NV_E4M3);
            const float2 f = __half22float2(__half2(r));
            const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * scale, f.y * scale);
            d[2 * i + h] = *reinterpret_cast<const uint32_t*>(&b);
        }
    }
}

template <int LAYOUT> __global__ void __launch_bounds__(PG_THREADS, 1) attn_paged_kernel(const PagedParams p) {
    constexpr bool F16 = LAYOUT == SMLA_LAYOUT_F16;
    constexpr bool PACKED = LAYOUT == SMLA_LAYOUT_V32 || LAYOUT == SMLA_LAYOUT_MODEL1;
    constexpr int CHUNKS = LAYOUT == SMLA_LAYOUT_MODEL1 ? 8 : 9;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* sm = smem_raw + (base - raw);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + GMISC_OFF + 4);
    const uint32_t abort_addr = base + GMISC_OFF + 4;
    auto bar = [&](int i) -> uint32_t { return base + GB_OFF + 8u * i; };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int part = blockIdx.x, row0 = (int)blockIdx.y * PG_ROWS;
    const int live = min(p.rows - row0, PG_ROWS);

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(GB_KFULL + i), PG_LD_WARPS / 2);
            mbar_init(bar(GB_KFREE + i), 1);
            mbar_init(bar(GB_SREADY + i), 1);
        }
        mbar_init(bar(GB_PREADY), PG_SM_WARPS);
        mbar_init(bar(GB_PVDONE), 1);
        mbar_init(bar(GB_QFREE), 1);
        *abort_flag = 0;
        for (int i = 0; i < 4; ++i) reinterpret_cast<volatile unsigned*>(sm + GN_OFF)[i] = 0u;
        mbar_init_fence();
    }
    if (warp == PG_MMA_WARP) { tmem_alloc(base + GMISC_OFF, 512); tmem_relinquish(); }
    grid_dep_wait();
    grid_dep_launch();

    // ---- the partition's part of the line: every thread sums the requests of its share, the block scans the sums
    long long* scan = reinterpret_cast<long long*>(sm + GW_OFF);
    const int per = (p.batch + PG_THREADS - 1) / PG_THREADS;
    const int r_lo = min(tid * per, p.batch), r_hi = min(r_lo + per, p.batch);
    long long sum = 0;
    for (int r = r_lo; r < r_hi; ++r) sum += paged_blocks(paged_length(p, r)) + PG_START;
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
    for (int w = 0; w <= PG_MMA_WARP; ++w) {
        if (w < warp) before += scan[w];
        total += scan[w];
    }
    const long long share = paged_share(total, p.num_parts), lo = min(part * share, total), hi = min(lo + share, total);
    if (before <= lo && lo < before + sum) {
        int r = r_lo;
        for (; r < r_hi - 1; ++r) {
            const int w = paged_blocks(paged_length(p, r)) + PG_START;
            if (lo < before + w) break;
            before += w;
        }
        scan[16] = before;
        *reinterpret_cast<int*>(scan + 17) = r;
    }
    __syncthreads();
    Pieces piece(lo, hi, lo < hi ? *reinterpret_cast<int*>(scan + 17) : p.batch, lo < hi ? scan[16] : 0);
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + GMISC_OFF);

    if (warp < PG_SM_WARPS) {
        // =================================================================== softmax + epilogue
        const int ra = 16 * warp + (lane >> 2), rb = ra + 8;      // the thread's query rows, columns 8 i + 2 (lane % 4) + {0, 1}
        const int quad = lane & 3;
        const uint32_t lane_addr = tmem + ((uint32_t)(warp * 32) << 16);
        const float c = p.sm_scale * LOG2E;
        float* factor = reinterpret_cast<float*>(sm + GA_OFF);
        unsigned* none = reinterpret_cast<unsigned*>(sm + GN_OFF);           // [2 stages] 64 bits
        const int cols = (live + 31) >> 5;                        // halves of 32 columns of O^T in use
        uint32_t it = 0;
        bool dead = false, stop = false;
        while (!stop && piece.next(p)) {
            const bool whole = piece.whole();
            if (row0 == 0 && tid == 0 && piece.b0 == 0) {
                const int last = piece.nb == 0 ? part : (int)((piece.start + PG_START + piece.nb - 1) / share);
                p.spans[piece.req] = make_int2(part, last);
            }
            // rows that query rows see: all of the request's, or up to the query's own
            const int hidden = p.causal ? p.query_len - 1 : 0;
            auto sees = [&](int r) { return p.causal ? min(max(piece.len - hidden + min(row0 + r, p.rows - 1) / p.num_heads, 0), piece.len) : piece.len; };
            const int see_a = sees(ra), see_b = sees(rb), see_least = sees(0);
            float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;
            for (int b = piece.b0; b < piece.b1; ++b, ++it) {
                if (!dead) dead = !mbar_wait_lean(bar(GB_SREADY + (it & 1)), (it >> 1) & 1u, abort_addr, WP_SREADY);
                uint32_t sv[32];
                float mx_a = -INFINITY, mx_b = -INFINITY;
                const int pos0 = b * 64;
                const bool tail = pos0 > see_least - 64;          // some row of the block is hidden from some query
                bool odd = false;
                if (!dead) {
                    tc_fence_after();
                    tmem_ld_16x256b_x8(lane_addr + GT_S + 64 * (it & 1), sv);
                    const unsigned long long valid = *reinterpret_cast<volatile unsigned long long*>(sm + GV_OFF + 8 * (it & 1));
                    tmem_wait_ld();
                    if (valid == ~0ull && !tail) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) sv[i] = __float_as_uint(__uint_as_float(sv[i]) * c);
                    } else {
                        unsigned bad[2] = {0u, 0u};
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const int col = 8 * (i >> 2) + 2 * quad + (i & 1);
                            const float x = __uint_as_float(sv[i]) * c;
                            const bool there = (valid >> col) & 1, seen = there && pos0 + col < ((i & 2) ? see_b : see_a);
                            if (there && !seen && !(fabsf(x) < INFINITY)) bad[col >> 5] |= 1u << (col & 31);
                            sv[i] = __float_as_uint(seen ? x : -INFINITY);
                        }
                        if (bad[0]) atomicOr(none + 2 * (it & 1), bad[0]);
                        if (bad[1]) atomicOr(none + 2 * (it & 1) + 1, bad[1]);
                        odd = (bad[0] | bad[1]) != 0u;
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        mx_a = fmaxf(mx_a, fmaxf(__uint_as_float(sv[i]), __uint_as_float(sv[i + 1])));
                        mx_b = fmaxf(mx_b, fmaxf(__uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3])));
                    }
#pragma unroll
                    for (int o = 1; o <= 2; o <<= 1) {
                        mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, o));
                        mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, o));
                    }
                }
                const bool grow_a = mx_a > m_a + PG_TAU, grow_b = mx_b > m_b + PG_TAU;      // false while a row has seen nothing
                const float al_a = grow_a ? ex2(m_a - mx_a) : 1.f, al_b = grow_b ? ex2(m_b - mx_b) : 1.f;
                if (quad == 0) { factor[ra] = al_a; factor[rb] = al_b; }
                if (named_bar_or(1, PG_SM_WARPS * 32, grow_a || grow_b || odd || dead || *abort_flag != 0)) {
                    // rare: a maximum grows, a hidden row is no number, or the CTA gives up
                    if (grow_a) { m_a = mx_a; l_a *= al_a; }
                    if (grow_b) { m_b = mx_b; l_b *= al_b; }
                    const unsigned long long hide = *reinterpret_cast<volatile unsigned long long*>(none + 2 * (it & 1));
                    if (b > piece.b0 && !dead) {
                        dead = !mbar_wait_lean(bar(GB_PVDONE), (it - 1) & 1u, abort_addr, WP_PVDONE);
                        tc_fence_after();
#pragma unroll 1
                        for (int k = 0; k < 8; ++k) {
                            if ((k & 1) >= cols) continue;
                            uint32_t o[32];
                            tmem_ld32(lane_addr + GT_O + 32 * k, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor[32 * (k & 1) + i]);
                            tmem_st32(lane_addr + GT_O + 32 * k, o);
                        }
                        tmem_wait_st();
                    }
                    if (hide != 0ull) {
                        // A row hidden from some query whose score is no number would reach that query through 0 x V: its values are
                        // taken out of the stage.  Queries that see it have a weight that is no number.
                        for (int i = tid; i < 64 * CHUNKS * 8; i += PG_SM_WARPS * 32) {
                            const int r = (i >> 3) & 63;
                            if ((hide >> r) & 1)
                                *reinterpret_cast<uint4*>(sm + GK_OFF + (it & 1) * G_STAGE + (i >> 9) * G_CHUNK + r * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
                        }
                    }
                    if (named_bar_or(1, PG_SM_WARPS * 32, dead || *abort_flag != 0)) { stop = true; break; }
                    if (tid == 0) *reinterpret_cast<volatile unsigned long long*>(none + 2 * (it & 1)) = 0ull;      // (next written two blocks from here)
                }
                const float ma = m_a == -INFINITY ? 0.f : m_a, mb = m_b == -INFINITY ? 0.f : m_b;
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float a0 = ex2(__uint_as_float(sv[4 * i]) - ma), a1 = ex2(__uint_as_float(sv[4 * i + 1]) - ma);
                    const float b0 = ex2(__uint_as_float(sv[4 * i + 2]) - mb), b1 = ex2(__uint_as_float(sv[4 * i + 3]) - mb);
                    l_a += a0 + a1;
                    l_b += b0 + b1;
                    w[2 * i] = pack_weights<F16>(a0, a1);
                    w[2 * i + 1] = pack_weights<F16>(b0, b1);
                }
                // the weights of the block before have been read
                if (it > 0 && !dead) dead = !mbar_wait_lean(bar(GB_PVDONE), (it - 1) & 1u, abort_addr, WP_PVDONE);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    *reinterpret_cast<uint32_t*>(sm + GP_OFF + gswz((uint32_t)ra, (uint32_t)i) + 4 * quad) = w[2 * i];
                    *reinterpret_cast<uint32_t*>(sm + GP_OFF + gswz((uint32_t)rb, (uint32_t)i) + 4 * quad) = w[2 * i + 1];
                }
                fence_proxy_async();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(GB_PREADY));
            }
            if (stop) break;
            // ---- epilogue
            if (piece.b1 > piece.b0 && !dead) dead = !mbar_wait_lean(bar(GB_PVDONE), (it - 1) & 1u, abort_addr, WP_PVDONE);
            tc_fence_after();
#pragma unroll
            for (int o = 1; o <= 2; o <<= 1) {
                l_a += __shfl_xor_sync(0xffffffffu, l_a, o);
                l_b += __shfl_xor_sync(0xffffffffu, l_b, o);
            }
            const size_t rec = whole ? (size_t)piece.req : (size_t)(2 * part + (piece.b0 == 0 ? 1 : 0));
            if (quad < 2) {                                       // one lane for each of the quad's rows
                const int r = quad == 0 ? ra : rb;
                const float l = quad == 0 ? l_a : l_b, m = quad == 0 ? m_a : m_b;
                float lse = l == 0.f ? NEG_BIG : log2f(l) + m, denom = l;
                if (r < live) {
                    if (whole && p.attn_sink != nullptr) {
                        const float sink2 = ld_in(p.attn_sink + (row0 + r) % p.num_heads) * LOG2E;
                        if (l != 0.f) denom += exp2f(sink2 - m);
                        lse = with_sink(lse, sink2);
                    }
                    (whole ? p.lse : p.lse_part)[rec * p.rows + row0 + r] = lse;
                }
                factor[r] = l == 0.f ? 0.f : 1.f / denom;         // 0: nothing is seen, or the sink takes all
            }
            if (named_bar_or(1, PG_SM_WARPS * 32, dead || *abort_flag != 0)) { stop = true; break; }
#pragma unroll 1
            for (int k = 0; k < 8; ++k) {
                if ((k & 1) >= cols) continue;
                uint32_t o[32];
                if (piece.b1 > piece.b0) tmem_ld32(lane_addr + GT_O + 32 * k, o);
                tmem_wait_ld();
                const size_t at = (rec * p.rows + row0 + 32 * (k & 1)) * D_V + 128 * (k >> 1) + 32 * warp + lane;
                const int n = min(live - 32 * (k & 1), 32);
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float f = factor[32 * (k & 1) + i], v = f == 0.f ? 0.f : __uint_as_float(o[i]) * f;
                    if (i < n) {
                        if (whole) static_cast<uint16_t*>(p.out)[at + (size_t)i * D_V] = out_bits<F16>(v);
                        else p.o_part[at + (size_t)i * D_V] = v;
                    }
                }
            }
            tc_fence_before();
            named_bar_sync(1, PG_SM_WARPS * 32);                  // the factors have been read
        }
    } else if (warp < PG_MMA_WARP) {
        // =================================================================== rows into the stages, and the queries
        const int stage = (warp - PG_SM_WARPS) >> 2, gw = (warp - PG_SM_WARPS) & 3;
        const uint32_t kst = GK_OFF + stage * G_STAGE;
        uint32_t it = 0, pieces = 0;
        bool ok = true;
        while (ok && piece.next(p)) {
            if (piece.b1 == piece.b0) continue;
            const int32_t* table = p.table + (int64_t)piece.req * p.table_stride;
            for (int b = piece.b0; b < piece.b1 && ok; ++b, ++it) {
                if ((it & 1) != (uint32_t)stage) continue;
                // where row r of the block lies: its page (null: no entry) and its place in there
                auto row_at = [&](int r, int& in) -> const uint8_t* {
                    const int pos = b * 64 + r;
                    in = 0;
                    if (pos >= piece.len) return nullptr;
                    const int j = pos / p.page_block_size, page = ld_in(table + j);
                    if (page < 0 || page >= p.num_pages) return nullptr;
                    in = pos - j * p.page_block_size;
                    return p.cache + (int64_t)page * p.page_stride;
                };
                unsigned bits = 0u;
                int in;
                if constexpr (!PACKED) {
                    const uint8_t* src[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        src[h] = row_at(16 * gw + 4 * h + (lane >> 3), in);
                        const unsigned v = __ballot_sync(0xffffffffu, src[h] != nullptr);
                        bits |= ((v & 1u) | ((v >> 7) & 2u) | ((v >> 14) & 4u) | ((v >> 21) & 8u)) << (4 * h);
                        if (src[h] != nullptr) src[h] += (int64_t)in * (2 * D_QK) + (lane & 7) * 16;
                    }
                    if (it >= 2) ok = mbar_wait_lean(bar(GB_KFREE + stage), ((it >> 1) - 1) & 1u, abort_addr, WP_KFREE);
                    if (!ok) break;
#pragma unroll
                    for (int ch = 0; ch < CHUNKS; ++ch) {
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            const bool there = src[h] != nullptr;
                            cp_async16(base + kst + ch * G_CHUNK + gswz((uint32_t)(16 * gw + 4 * h + (lane >> 3)), lane & 7),
                                       there ? src[h] + ch * 128 : p.q, there ? 16u : 0u);
                        }
                    }
                } else {
                    constexpr int NOPE = LAYOUT == SMLA_LAYOUT_V32 ? D_NOPE : 448;
                    constexpr int ROPE_AT = LAYOUT == SMLA_LAYOUT_V32 ? ROPE_OFF : 448;
                    const uint8_t* mine = row_at(16 * gw + (lane & 15), in);       // lane i: row i % 16 of the warp
                    bits = __ballot_sync(0xffffffffu, mine != nullptr) & 0xffffu;
                    uint2 sc8 = make_uint2(0u, 0u);
                    unsigned long long at = 0ull;
                    if (mine != nullptr) {
                        if (LAYOUT == SMLA_LAYOUT_MODEL1)
                            sc8 = ld_in(reinterpret_cast<const uint2*>(mine + (int64_t)p.page_block_size * SMLA_M1_DATA_BYTES + (int64_t)in * 8));
                        at = reinterpret_cast<unsigned long long>(mine + (int64_t)in * (LAYOUT == SMLA_LAYOUT_V32 ? ROW_BYTES : SMLA_M1_DATA_BYTES));
                    }
                    uint4 nope[16], rope[4];
                    float scale[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint8_t* src = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, at, i));
                        nope[i] = make_uint4(0, 0, 0, 0);
                        scale[i] = 0.f;
                        if (src != nullptr && lane < NOPE / 16) nope[i] = ld_in_once(reinterpret_cast<const uint4*>(src) + lane);
                        if (LAYOUT == SMLA_LAYOUT_V32 && src != nullptr) scale[i] = ld_in(reinterpret_cast<const float*>(src + SCALE_OFF) + (lane >> 3));
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint8_t* src = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, at, 4 * u + (lane >> 3)));
                        rope[u] = make_uint4(0, 0, 0, 0);
                        if (src != nullptr) rope[u] = ld_in_once(reinterpret_cast<const uint4*>(src + ROPE_AT) + (lane & 7));
                    }
                    if (it >= 2) ok = mbar_wait_lean(bar(GB_KFREE + stage), ((it >> 1) - 1) & 1u, abort_addr, WP_KFREE);
                    if (!ok) break;
                    const uint32_t chunk = kst + (lane >> 2) * G_CHUNK;
                    const bool swap = (lane & 4) != 0;           // neighbouring chunks store their two pieces in opposite order: no bank conflicts
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint32_t r = (uint32_t)(16 * gw + i), pc = 2u * (lane & 3);
                        float f = scale[i];
                        if (LAYOUT == SMLA_LAYOUT_MODEL1) {
                            const uint32_t w0 = __shfl_sync(0xffffffffu, sc8.x, i), w1 = __shfl_sync(0xffffffffu, sc8.y, i);
                            f = __uint_as_float(((((lane & 16) ? w1 : w0) >> (8 * ((lane >> 2) & 3))) & 0xffu) << 23);
                        }
                        uint32_t d[8];
                        dequant16(nope[i], f, d);
                        const uint4 lo4 = make_uint4(d[0], d[1], d[2], d[3]), hi4 = make_uint4(d[4], d[5], d[6], d[7]);
                        if (lane < NOPE / 16) {
                            *reinterpret_cast<uint4*>(sm + chunk + gswz(r, pc + (swap ? 1u : 0u))) = swap ? hi4 : lo4;
                            *reinterpret_cast<uint4*>(sm + chunk + gswz(r, pc + (swap ? 0u : 1u))) = swap ? lo4 : hi4;
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        *reinterpret_cast<uint4*>(sm + kst + (CHUNKS - 1) * G_CHUNK + gswz((uint32_t)(16 * gw + 4 * u + (lane >> 3)), lane & 7)) = rope[u];
                }
                if (b == piece.b0) {                              // the piece's queries come with its first block
                    if (pieces > 0) ok = mbar_wait_lean(bar(GB_QFREE), (pieces - 1) & 1u, abort_addr, WP_QFREE);
                    if (!ok) break;
                    const uint8_t* q = p.q + ((size_t)piece.req * p.rows + row0) * (CHUNKS * 128);
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const int r = 16 * gw + 4 * h + (lane >> 3);
                        const bool there = r < live;
                        const uint8_t* at = there ? q + (size_t)r * (CHUNKS * 128) + (lane & 7) * 16 : p.q;
#pragma unroll
                        for (int ch = 0; ch < CHUNKS; ++ch)
                            cp_async16(base + GQ_OFF + ch * G_CHUNK + gswz((uint32_t)r, lane & 7), at + (there ? ch * 128 : 0), there ? 16u : 0u);
                    }
                }
                cp_async_wait_all();
                if (lane == 0) *reinterpret_cast<volatile uint16_t*>(sm + GV_OFF + 8 * stage + 2 * gw) = (uint16_t)bits;
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(GB_KFULL + stage));
            }
            ++pieces;
        }
    } else {
        // =================================================================== MMA issue
        const uint32_t idesc_s = instr_desc(F16 ? FMT_F16 : FMT_BF16, F16 ? FMT_F16 : FMT_BF16, false, false, 64, 64);
        const uint32_t idesc_o = instr_desc(F16 ? FMT_F16 : FMT_BF16, F16 ? FMT_F16 : FMT_BF16, true, false, 128, (uint32_t)((live + 15) & ~15));
        const uint32_t q_lo = desc_lo(base + GQ_OFF, 16), k_lo = desc_lo(base + GK_OFF, 16);
        const uint32_t v_lo = desc_lo(base + GK_OFF, G_CHUNK), p_lo = desc_lo(base + GP_OFF, 16);      // V MN-major: the next 64 dims lie a chunk further
        uint32_t scored = 0, done = 0, firsts = 0;                // blocks whose scores / whose P.V have been issued; bit i: block i % 2 is its piece's first
        bool ok = true, have = false;
        int b = 0;
        auto advance = [&]() {                                    // to the next block
            if (have && ++b < piece.b1) return;
            do { have = piece.next(p); } while (have && piece.b1 == piece.b0);
            b = piece.b0;
        };
        advance();
        while (ok && (have || done < scored)) {
            // scores run at most one block ahead of P.V (their buffer, and the order in which stages become free)
            const bool may_score = have && scored - done <= 1;
            bool score = false;
            if (may_score && scored == done) {
                ok = mbar_wait_lean(bar(GB_KFULL + (scored & 1)), (scored >> 1) & 1u, abort_addr, WP_KFULL);
                score = true;
            } else {
                // whichever is ready first: the next block's rows or this one's weights
                uint32_t left = 1u << 26;
                while (true) {
                    if (may_score && __all_sync(0xffffffffu, mbar_test(bar(GB_KFULL + (scored & 1)), (scored >> 1) & 1u))) { score = true; break; }
                    if (__all_sync(0xffffffffu, mbar_test(bar(GB_PREADY), done & 1u))) break;
                    if (--left == 0u) { ok = mbar_wait_lean(bar(GB_PREADY), done & 1u, abort_addr, WP_PREADY); break; }
                }
            }
            if (!ok) break;
            tc_fence_after();
            if (score) {
                const uint32_t st = scored & 1;
                firsts = (firsts & ~(1u << st)) | ((b == piece.b0 ? 1u : 0u) << st);
                const bool last = b + 1 == piece.b1;
                if (elect_one()) {
#pragma unroll 1
                    for (int ch = 0; ch < CHUNKS; ++ch) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_f16(tmem + GT_S + 64 * st, make_desc(q_lo + ((ch * G_CHUNK + k * 32) >> 4), G_DESC_HI),
                                    make_desc(k_lo + ((st * G_STAGE + ch * G_CHUNK + k * 32) >> 4), G_DESC_HI), idesc_s, (ch | k) != 0);
                    }
                    tc_commit(bar(GB_SREADY + st));
                    if (last) tc_commit(bar(GB_QFREE));
                }
                __syncwarp();
                ++scored;
                advance();
            } else {
                const uint32_t st = done & 1;
                const bool first = (firsts >> st) & 1u;
                if (elect_one()) {
#pragma unroll 1
                    for (int k = 0; k < 4; ++k) {
#pragma unroll
                        for (int d = 0; d < 4; ++d)
                            mma_f16(tmem + GT_O + 64 * d, make_desc(v_lo + ((st * G_STAGE + 2 * d * G_CHUNK + k * 2048) >> 4), G_DESC_HI),
                                    make_desc(p_lo + ((k * 32) >> 4), G_DESC_HI), idesc_o, !first || k != 0);
                    }
                    tc_commit(bar(GB_KFREE + st));
                    tc_commit(bar(GB_PVDONE));
                }
                __syncwarp();
                ++done;
            }
        }
    }

    if (*abort_flag != 0) {        // a wait gave up: MMAs may still be in flight; give them time to finish
        const long long t0 = clock64();
        while (clock64() - t0 < 200000) { }
    }
    cp_async_wait_all();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *abort_flag != 0 && p.status != nullptr) {
        atomicCAS(p.status, 0, *abort_flag);
        atomicAdd(p.status + 1, 1);
        p.status[2] = blockIdx.x;
    }
    if (warp == PG_MMA_WARP) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

// One warp per query row of a request: joins what its partitions left, in their order.  Requests within one partition are done.
template <bool F16> __global__ void __launch_bounds__(256) paged_combine_kernel(const PagedParams p) {
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31;
    const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (id >= (int64_t)p.batch * p.rows) return;
    const int req = (int)(id / p.rows), row = (int)(id - (int64_t)req * p.rows);
    const uint2 span = ld_in(reinterpret_cast<const uint2*>(p.spans + req));
    const int c0 = (int)span.x, n = (int)span.y - c0 + 1;
    if (n <= 1) return;
    auto record = [&](int s) { return (size_t)(s == 0 ? 2 * c0 + 1 : 2 * (c0 + s)) * p.rows + row; };
    float mx = NEG_BIG, sum = 0.f;
    for (int s = lane; s < n; s += 32) mx = fmaxf(mx, ld_in(p.lse_part + record(s)));
    mx = warp_max(mx);
    for (int s = lane; s < n; s += 32) {
        const float v = ld_in(p.lse_part + record(s));
        sum += v == NEG_BIG ? 0.f : exp2f(v - mx);
    }
    sum = warp_sum(sum);
    float lse = sum == 0.f ? NEG_BIG : log2f(sum) + mx, denom = sum;
    if (p.attn_sink != nullptr) {
        const float sink2 = ld_in(p.attn_sink + row % p.num_heads) * LOG2E;
        if (sum != 0.f) denom += exp2f(sink2 - mx);
        lse = with_sink(lse, sink2);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / denom;
    float4 acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < n; ++s) {
        const size_t r = record(s);
        const float v = ld_in(p.lse_part + r), w = v == NEG_BIG ? 0.f : exp2f(v - mx) * inv;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 x = ld_in_once(reinterpret_cast<const float4*>(p.o_part + r * D_V + i * 128 + lane * 4));
            acc[i].x += w * x.x; acc[i].y += w * x.y; acc[i].z += w * x.z; acc[i].w += w * x.w;
        }
    }
    if (lane == 0) p.lse[id] = lse;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint2 v = make_uint2(pack_weights<F16>(acc[i].x, acc[i].y), pack_weights<F16>(acc[i].z, acc[i].w));
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + (size_t)id * D_V + i * 128 + lane * 4) = v;
    }
}

}  // namespace

int paged_parts(int batch, int rows, int pages_per_request, int page_block_size, int num_parts) {
    if (num_parts > 0) return num_parts;
    const int sms = smla_num_sms();
    if (sms < 1) return 0;
    const int groups = (rows + PG_ROWS - 1) / PG_ROWS, most = sms / groups > 0 ? sms / groups : 1;
    const long long blocks = ((long long)pages_per_request * page_block_size + 63) / 64;
    const long long worth = (batch * (blocks + PG_START) + PG_START + PG_LEAST - 1) / (PG_START + PG_LEAST);
    return worth < most ? (int)(worth > 0 ? worth : 1) : most;
}

int launch_attn_paged(const PagedParams& p, int layout, cudaStream_t stream) {
    typedef void (*Kernel)(const PagedParams);
    static const Kernel kernels[4] = {attn_paged_kernel<SMLA_LAYOUT_V32>, attn_paged_kernel<SMLA_LAYOUT_MODEL1>, attn_paged_kernel<SMLA_LAYOUT_BF16>,
                                      attn_paged_kernel<SMLA_LAYOUT_F16>};
    static std::atomic<bool> attr_set[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return set_error(SMLA_E_SHAPE, "attn_paged_kernel: device ordinal %d not supported", dev);
    if (!attr_set[dev]) {
        for (const Kernel k : kernels) {
            const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)G_SMEM);
            if (e != cudaSuccess) return set_error((int)e, "attn_paged_kernel: cannot reserve %u bytes of shared memory: %s", G_SMEM, cudaGetErrorString(e));
        }
        attr_set[dev] = true;
    }
    const Kernel kernel = layout == SMLA_LAYOUT_V32      ? attn_paged_kernel<SMLA_LAYOUT_V32>
                          : layout == SMLA_LAYOUT_MODEL1 ? attn_paged_kernel<SMLA_LAYOUT_MODEL1>
                          : layout == SMLA_LAYOUT_BF16   ? attn_paged_kernel<SMLA_LAYOUT_BF16>
                                                         : attn_paged_kernel<SMLA_LAYOUT_F16>;
    launch_dependent(kernel, dim3(p.num_parts, (p.rows + PG_ROWS - 1) / PG_ROWS), dim3(PG_THREADS), G_SMEM, stream, p);
    if (int e = check_launch("attn_paged_kernel")) return e;
    if (p.num_parts == 1) return 0;                // every request is whole
    const int64_t blocks = ((int64_t)p.batch * p.rows + 7) / 8;
    launch_dependent(layout == SMLA_LAYOUT_F16 ? paged_combine_kernel<true> : paged_combine_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return check_launch("paged_combine_kernel");
}

}  // namespace smla
