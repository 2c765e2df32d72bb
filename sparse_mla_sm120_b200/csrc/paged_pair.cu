// Attention over a block table of more than 64 query rows per request, 16-bit rows: attn_paged_kernel's work on a pair of SMs
// (tcgen05.mma.cta_group::2), 128 query rows and blocks of 128 cache rows.
//
// The formulas, the line of blocks that partitions cut, records and merge are those of paged.cu.  A cluster of two CTAs has 128 query rows, 64
// each, and every MMA runs over the pair with M = 128:
//   * S = Q . K^T: A = the CTA's queries, B = the 64 of the block's 128 rows that it has brought in (9 chunks of 64 dims, K-major);
//     lanes 0-63 of a CTA's tensor memory get its query rows against rows 0-63 of the block, lanes 64-127 against rows 64-127;
//   * O += P . V: A = the CTA's weights [64 x 128 rows], B = dims [256 r, +256) of all 128 rows in CTA r (MN-major), N = 256 in two
//     products; lanes 0-63 get dims 0-255, lanes 64-127 dims 256-511: 256 columns of tensor memory.
// Why a pair: operands of 64 rows keep the tensor core waiting for shared memory (M = N = 64: 40.6 cycles of the 16 that the arithmetic
// takes; measured over 36 products in a row).  Over the pair M = N = 128 takes 41.8 for four times the products of one of the
// CTAs' 64 x 64, M = 128 and N = 256 70: 2630 cycles per 128 x 128 where two CTAs of paged.cu take 4600.
// What it costs: V comes in beside K (64 KB next to 72 KB per CTA and block, from L2), since a CTA has other dims of other rows in V than
// in K, and the two fill shared memory: one stage of each, freed and filled again in parts while the products of the others run.
//
// What bounds it: memory and the chain K -> scores -> softmax -> P.V about equally, 3900 to 4300 cycles per block (136 KB per CTA from L2, 147 KB per
// pair from HBM: 5 TB/s), and what a request costs besides: 15000 cycles before the first scores, 9000 for an epilogue.
// 64 requests of up to 8192 rows, 128 heads: 114 to 118 us from one B200 to another (3.0 TB/s, 700 TFLOP/s); one of 131072: 58 us, of which the merge takes 9.
// The steps (us, both cases): as two CTAs of paged.cu 149.6, 72.7; first version 129.9, 65.8; the even CTA's barriers take the bytes of both,
// weights handed over by halves, epilogue through shared memory, 16 warps of 128 registers (16 bytes of them spilled) 116.4, 60.1.  Measured and not
// kept: a barrier per chunk of K (400 cycles each to issue: 135.4), V by two warps (141.5), 20 warps that trade registers (131.1).
//
// Warps: 0-7 softmax and epilogue (thread = one query row x 32 rows of a block), 8 and 9 bring in K and the queries, 10-13 V (64 rows x
// 128 dims each), 14 issues the score products, 15 those with V: both in the even CTA, in the odd one 15 passes on that its V has landed.
// Every wait is bounded; a wait that gives up records a code in status[] and the CTA drains and exits.
#include "paged_common.cuh"
#include "rows_map.cuh"

namespace smla {

namespace {

constexpr int PP_TILE = 128;                      // cache rows of a block, and query rows of a pair
constexpr int PP_SM_WARPS = 8, PP_K0 = 8, PP_V0 = 10, PP_S_WARP = 14, PP_PV_WARP = 15, PP_WARPS = 16, PP_THREADS = PP_WARPS * 32;
constexpr int PP_CHUNKS = 9;

constexpr uint32_t PPQ_OFF = 0;
constexpr uint32_t PPK_OFF = PPQ_OFF + PP_CHUNKS * G_CHUNK;
constexpr uint32_t PPV_OFF = PPK_OFF + PP_CHUNKS * G_CHUNK;   // [2 halves of the block's rows][4 chunks of 64 dims]
constexpr uint32_t PPP_OFF = PPV_OFF + 8 * G_CHUNK;           // weights: [2 halves of the block's rows][64 query rows][64]
constexpr uint32_t PPX_OFF = PPP_OFF + 2 * G_CHUNK;           // [4][64] fp32: maxima, then sums, of the four threads of a query row
constexpr uint32_t PPW_OFF = PPX_OFF + 4 * 64 * 4;            // schedule
constexpr uint32_t PPY_OFF = PPW_OFF + 24 * 8;                // which of a block's rows are there, [8 blocks] 128 bits
constexpr uint32_t PPB_OFF = PPY_OFF + 8 * 16;
// Barriers; those with a P collect arrivals of both CTAs and are used in the even one only.
constexpr int PB_KFULLP = 0, PB_KFREE = PB_KFULLP + 4, PB_VFULL = PB_KFREE + 4, PB_VPEERP = PB_VFULL + 2, PB_VFREE = PB_VPEERP + 2,
              PB_SREADY = PB_VFREE + 2, PB_SFREEP = PB_SREADY + 2, PB_PREADYP = PB_SFREEP + 2, PB_QFREE = PB_PREADYP + 2,
              PB_N = PB_QFREE + 1;
constexpr uint32_t PPMISC_OFF = PPB_OFF + PB_N * 8;
constexpr uint32_t PP_SMEM = (PPMISC_OFF + 8 + 15) / 16 * 16 + 1024;
static_assert(PP_SMEM <= 227 * 1024, "shared memory budget");
static_assert(PPY_OFF % 16 == 0 && PPB_OFF % 8 == 0 && PPMISC_OFF % 8 == 0, "alignment");

constexpr uint32_t PPT_O = 0, PPT_S = 256;        // tensor memory: O 2 x 128 columns, two score buffers of 64
constexpr uint32_t PP_DESC_HI = desc_hi(1024, (uint32_t)SWIZZLE_128B);

enum { WQ_KFULL = 91, WQ_KFREE = 93, WQ_VFULL = 94, WQ_VPEER = 95, WQ_VFREE = 96, WQ_SREADY = 97, WQ_SFREE = 98, WQ_PREADY = 99,
       WQ_QFREE = 101 };

// The block's rows that are there and the pages of their copies: lane i sees to copies i, i + 32, i + 64 and i + 96 of `rows` rows each.
struct BlockPlaces {
    int page[4], in[4], q_row;
    uint32_t valid[4];                            // the same in all lanes
    bool have, first;                             // there is such a block; it is the first of its piece
};

// Walks a partition's blocks.
struct BlockWalk {
    Pieces<PP_TILE> piece;
    int b;
    bool more;
    __device__ __forceinline__ BlockWalk(const PagedParams& p, const Pieces<PP_TILE>& first) : piece(first), b(-1) { more = piece.next(p); }
    __device__ __forceinline__ void look_up(const PagedParams& p, int row0, BlockPlaces& w) {
        w.have = more;
        if (!more) return;
        if (b < 0) {
            while (piece.b1 == piece.b0) {
                if (!piece.next(p)) { w.have = more = false; return; }
            }
            b = piece.b0;
        }
        w.first = b == piece.b0;
        w.q_row = piece.req * p.rows + row0;
        const int lane = threadIdx.x & 31, rows = p.copy_rows, copies = PP_TILE / rows;
        uint32_t mine[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = lane + 32 * u;
            w.page[u] = -1;
            w.in[u] = 0;
            if (i >= copies) continue;
            const int pos = b * PP_TILE + i * rows;
            if (pos >= piece.len) continue;
            const int j = pos / p.page_block_size, e = ld_in(p.table + (int64_t)piece.req * p.table_stride + j);
            if (e < 0 || e >= p.num_pages) continue;
            w.page[u] = e;
            w.in[u] = pos - j * p.page_block_size;
            // rows [i rows, + k) of the block
            const int k = min(piece.len - pos, rows), at = i * rows;
            if (rows >= 32) {
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const int n = min(max(at + k - 32 * v, 0), 32);
                    if (32 * v >= at && n > 0) mine[v] |= n == 32 ? ~0u : (1u << n) - 1u;
                }
            } else {
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    if ((at >> 5) == v) mine[v] |= ((1u << k) - 1u) << (at & 31);
            }
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) w.valid[v] = __reduce_or_sync(0xffffffffu, mine[v]);
        if (++b == piece.b1) {
            more = piece.next(p);
            b = -1;
        }
    }
};

// one(copy's number, its page, its first row in the page) for copies [i0, i1) that are there, in one lane with operands that are the same in all.
template <class F> __device__ __forceinline__ void each_copy(const BlockPlaces& w, int i0, int i1, F&& one) {
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
        const int u = i >> 5;
        const int pg = u == 0 ? w.page[0] : u == 1 ? w.page[1] : u == 2 ? w.page[2] : w.page[3], in = u == 0 ? w.in[0] : u == 1 ? w.in[1] : u == 2 ? w.in[2] : w.in[3];
        const int e = __shfl_sync(0xffffffffu, pg, i & 31), y = __shfl_sync(0xffffffffu, in, i & 31);
        if (e >= 0 && elect_one()) one(i, e, y);
    }
    __syncwarp();
}
// How many of copies [i0, i1) there are.
__device__ __forceinline__ uint32_t copies_of(const BlockPlaces& w, int i0, int i1) {
    uint32_t n = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int i = (int)(threadIdx.x & 31) + 32 * u;
        n += (uint32_t)__popc(__ballot_sync(0xffffffffu, w.page[u] >= 0 && i >= i0 && i < i1));
    }
    return n;
}

template <bool F16> __global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PP_THREADS, 1)
attn_paged_pair_kernel(const PagedParams p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* sm = smem_raw + (base - raw);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + PPMISC_OFF + 4);
    const uint32_t abort_addr = base + PPMISC_OFF + 4;
    auto bar = [&](int i) -> uint32_t { return base + PPB_OFF + 8u * i; };
    auto barp = [&](int i) -> uint32_t { return mapa_shared(bar(i), 0); };     // the even CTA's
    auto commit_both = [&](int i) {
        tc_commit_pair(bar(i));
        tc_commit_pair(mapa_shared(bar(i), 1));
    };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank();
    const int part = blockIdx.x >> 1, group0 = (int)blockIdx.y * PP_TILE, row0 = group0 + 64 * (int)rank;
    const int live = min(max(p.rows - row0, 0), 64);

    if (tid == 0) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(bar(PB_KFULLP + i), 2);                     // + the bytes of both CTAs' rows
            mbar_init(bar(PB_KFREE + i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(PB_VFULL + i), 2);
            mbar_init(bar(PB_VPEERP + i), 1);
            mbar_init(bar(PB_VFREE + i), 1);
            mbar_init(bar(PB_SREADY + i), 1);
            mbar_init(bar(PB_SFREEP + i), 2 * PP_SM_WARPS);
            mbar_init(bar(PB_PREADYP + i), PP_SM_WARPS);          // half of the softmax warps of both CTAs: the weights of half of a block's rows
        }
        mbar_init(bar(PB_QFREE), 1);
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == PP_S_WARP) { tmem_alloc_pair(base + PPMISC_OFF, 512); tmem_relinquish_pair(); }
    cluster_sync_all();          // the partner's barriers exist before anything arrives on them
    grid_dep_wait();
    grid_dep_launch();
    Pieces<PP_TILE> piece = partition_of<PP_TILE>(p, part, reinterpret_cast<long long*>(sm + PPW_OFF), PP_WARPS);
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + PPMISC_OFF);

    if (warp < PP_SM_WARPS) {
        // =================================================================== softmax + epilogue
        const int quarter = warp & 3, ch = warp >> 2, grp = quarter & 1, thalf = quarter >> 1;
        const int hrow = 32 * grp + lane, xpart = 2 * thalf + ch;
        const int col0 = 64 * thalf + 32 * ch;                    // the thread's rows of a block: [col0, + 32)
        const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
        // The sign of the softmax scale goes into the scores.  Never 0: rows that are not seen have scores of -inf, and -inf times 0 would be no
        // number; the smallest normal number takes scores of up to 2^100 to nothing.  (A scale that is no number stays none.)
        const float c = p.sm_scale == p.sm_scale ? fmaxf(fabsf(p.sm_scale * LOG2E), 0x1p-126f) : p.sm_scale;
        const bool negative = p.sm_scale < 0.f;
        float* xch = reinterpret_cast<float*>(sm + PPX_OFF);
        const uint32_t s_free = barp(PB_SFREEP), p_ready = barp(PB_PREADYP + thalf);
        uint32_t it = 0;
        bool dead = false, stop = false;
        while (!stop && piece.next(p)) {
            const bool whole = piece.whole();
            if (group0 == 0 && rank == 0 && tid == 0 && piece.b0 == 0) piece.write_span(p, part, reinterpret_cast<long long*>(sm + PPW_OFF)[20]);
            const int see = paged_sees(p, piece.len, row0 + hrow);
            const int see_least = paged_sees(p, piece.len, group0);       // of the pair's query rows
            float m = -INFINITY, l = 0.f;
            for (int b = piece.b0; b < piece.b1; ++b, ++it) {
                const uint32_t st = it & 1;
                if (!dead) dead = !mbar_wait_lean(bar(PB_SREADY + st), (it >> 1) & 1u, abort_addr, WQ_SREADY);
                uint32_t sv[32];
                float mx = -INFINITY;
                const int pos0 = b * PP_TILE;
                bool plain = true;                                // all rows are there and seen by all query rows
                const uint4 valid = *reinterpret_cast<const uint4*>(sm + PPY_OFF + 16 * (it & 7));
                if (!dead) {
                    tc_fence_after();
                    tmem_ld32(lane_addr + PPT_S + 64 * st + 32 * ch, sv);
                    plain = (valid.x & valid.y & valid.z & valid.w) == ~0u && pos0 <= see_least - PP_TILE;
                    tmem_wait_ld();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_remote(s_free + 8 * st);
                    if (negative) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) sv[i] ^= 0x80000000u;
                    }
                    if (!plain) {
                        uint32_t seen = col0 < 32 ? valid.x : col0 < 64 ? valid.y : col0 < 96 ? valid.z : valid.w;
                        const int n = see - pos0 - col0;          // of the thread's 32 rows, those before the query's last
                        seen = n <= 0 ? 0u : n < 32 ? seen & ((1u << n) - 1u) : seen;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!((seen >> i) & 1u)) sv[i] = 0xff800000u;
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 2) mx = fmaxf(fmaxf(mx, __uint_as_float(sv[i])), __uint_as_float(sv[i + 1]));
                    mx *= c;
                }
                // The four threads of a query row (in the four warps of a barrier) exchange their maxima only when one of the barrier's rows has
                // outgrown its running maximum: rare after a request's first blocks.
                if (named_bar_or(1 + grp, 128, mx > m + PG_TAU || dead)) {
                    xch[64 * xpart + hrow] = mx;
                    if (named_bar_or(1 + grp, 128, dead || *abort_flag != 0)) { stop = true; break; }
                    const float all = fmaxf(fmaxf(xch[hrow], xch[64 + hrow]), fmaxf(xch[128 + hrow], xch[192 + hrow]));
                    float al = 1.f;
                    if (all > m + PG_TAU) { al = ex2(m - all); m = all; l *= al; }
                    if (b > piece.b0 && __any_sync(0xffffffffu, al != 1.f)) {
                        // All products of the block before.  (A parity tells a phase from its neighbours only: the phase before this one
                        // is known to be over, for the thalf 1 warps waited for it ahead of the barriers above.)
                        dead = !mbar_wait_lean(bar(PB_VFREE + 1), (it - 1) & 1u, abort_addr, WQ_VFREE);
                        if (!dead) {
                            tc_fence_after();
#pragma unroll 1
                            for (int d = 0; d < 128; d += 16) {
                                const uint32_t at = lane_addr + PPT_O + 128 * ch + d;
                                uint32_t o[16];
                                tmem_ld16(at, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * al);
                                tmem_st16(at, o);
                            }
                            tmem_wait_st();
                        }
                    }
                    // The products of either half of the block's rows add to all lanes of O and begin when the warps of that half have
                    // arrived: none of them does before all four have rescaled.
                    tc_fence_before();
                    if (named_bar_or(1 + grp, 128, dead)) { stop = true; break; }
                    tc_fence_after();
                }
                const float mm = m == -INFINITY ? 0.f : -m;
                // s c - m in one rounding is off from the rounded maximum by as much as that was rounded: harmless (it stands in all weights and in
                // their sum) while that is less than a step of an exponent, but not where scores have steps of hundreds.
                float cc = c;
                if (fabsf(mm) >= 0x1p24f) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) sv[i] = __float_as_uint(__uint_as_float(sv[i]) * c);
                    cc = 1.f;
                }
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float a = ex2(fmaf(__uint_as_float(sv[2 * i]), cc, mm)), e = ex2(fmaf(__uint_as_float(sv[2 * i + 1]), cc, mm));
                    l += a + e;
                    w[i] = pack_weights<F16>(a, e);
                }
                // The weights of the block before have been read.  (Each half of a block's rows has its own hand-over, so that the weights of one are
                // stored while the products of the other run: a second buffer does not fit.)
                if (it > 0 && !dead) dead = !mbar_wait_lean(bar(PB_VFREE + thalf), (it - 1) & 1u, abort_addr, WQ_VFREE);
                if (!plain && !dead) {
                    // Rows that are not there, and values that are no numbers in rows hidden from some query, would reach queries through
                    // 0 x V: they are taken out of the stage.  (A query that sees such a row has a weight that is no number.)
                    dead = !mbar_wait_lean(bar(PB_VFULL + thalf), it & 1u, abort_addr, WQ_VFULL);
                    if (!dead) {
                        const uint32_t there0 = thalf ? valid.z : valid.x, there1 = thalf ? valid.w : valid.y;
#pragma unroll 1
                        for (int i = (2 * grp + ch) * 32 + lane; i < 64 * 32; i += 128) {
                            const int r = (i >> 3) & 63;
                            uint4* at = reinterpret_cast<uint4*>(sm + PPV_OFF + (4 * thalf + (i >> 9)) * G_CHUNK + r * 128 + (i & 7) * 16);
                            if (!(((r & 32 ? there1 : there0) >> (r & 31)) & 1u)) {
                                *at = make_uint4(0, 0, 0, 0);
                            } else if (pos0 + 64 * thalf + r >= see_least) {
                                *at = numbers_only<F16>(*at);
                            }
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<uint4*>(sm + PPP_OFF + thalf * G_CHUNK + gswz((uint32_t)hrow, (uint32_t)(4 * ch + i))) =
                        make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                fence_proxy_async();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_remote(p_ready);
            }
            if (stop) break;
            // ---- epilogue
            // Behind this barrier the maxima have been read, and the thalf 1 warps have waited for half 1 of the block before the last: the
            // parity that is asked for next is the last block's.
            if (named_bar_or(1 + grp, 128, dead || *abort_flag != 0)) { stop = true; break; }
            if (piece.b1 > piece.b0) dead = !mbar_wait_lean(bar(PB_VFREE + 1), (it - 1) & 1u, abort_addr, WQ_VFREE);
            xch[64 * xpart + hrow] = l;
            if (named_bar_or(1 + grp, 128, dead)) { stop = true; break; }
            tc_fence_after();
            l = (xch[hrow] + xch[64 + hrow]) + (xch[128 + hrow] + xch[192 + hrow]);
            const size_t rec = whole ? (size_t)piece.req : (size_t)(2 * part + (piece.b0 == 0 ? 1 : 0));
            const size_t row = rec * p.rows + row0 + hrow;
            float lse = l == 0.f ? (whole ? NEG_BIG : NO_RECORD) : log2f(l) + m, denom = l;
            if (whole && p.attn_sink != nullptr && hrow < live) {
                const float sink2 = ld_in(p.attn_sink + (row0 + hrow) % p.num_heads) * LOG2E;
                if (l != 0.f) denom += exp2f(sink2 - m);
                lse = with_sink(lse, sink2);
            }
            if (xpart == 0 && hrow < live) (whole ? p.lse : p.lse_part)[row] = lse;
            const float f = l == 0.f ? 0.f : 1.f / denom;         // 0: nothing is seen, or the sink takes all
            // 32 dims of each of the warp's 32 query rows at a time, through the weights' place in shared memory, so that four (16-bit) or eight
            // lanes write a row's neighbouring bytes.  Of the place, the two warps of a quarter have what they later write weights to: after
            // the next barrier of both.
            uint8_t* stage = sm + PPP_OFF + thalf * G_CHUNK + grp * 4096 + ch * 2048;
            const int first_row = row0 + 32 * grp, mine = live - 32 * grp;
#pragma unroll 1
            for (int d = 0; d < 128; d += 32) {
                uint32_t o[32];
                if (piece.b1 > piece.b0) tmem_ld32(lane_addr + PPT_O + 128 * ch + d, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = f == 0.f ? 0u : __float_as_uint(__uint_as_float(o[i]) * f);
                const size_t at = (rec * p.rows + first_row) * D_V + 256 * thalf + 128 * ch + d;
                if (whole) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<uint4*>(stage + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) =
                            make_uint4(pack_weights<F16>(__uint_as_float(o[8 * i]), __uint_as_float(o[8 * i + 1])), pack_weights<F16>(__uint_as_float(o[8 * i + 2]), __uint_as_float(o[8 * i + 3])),
                                       pack_weights<F16>(__uint_as_float(o[8 * i + 4]), __uint_as_float(o[8 * i + 5])), pack_weights<F16>(__uint_as_float(o[8 * i + 6]), __uint_as_float(o[8 * i + 7])));
                    __syncwarp();
                    uint8_t* dst = reinterpret_cast<uint8_t*>(static_cast<uint16_t*>(p.out) + at) + (lane & 3) * 16;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int r = 8 * j + (lane >> 2);
                        const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
                        if (r < mine) *reinterpret_cast<uint4*>(dst + (size_t)r * (2 * D_V)) = v;
                    }
                    __syncwarp();
                } else {
                    uint8_t* dst = reinterpret_cast<uint8_t*>(p.o_part + at) + (lane & 7) * 16;
#pragma unroll
                    for (int pass = 0; pass < 2; ++pass) {
                        if ((lane >> 4) == pass) {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                *reinterpret_cast<uint4*>(stage + gswz((uint32_t)lane & 15u, (uint32_t)i)) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        }
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int r = 4 * j + (lane >> 3);
                            const uint4 v = *reinterpret_cast<const uint4*>(stage + gswz((uint32_t)r, (uint32_t)lane & 7u));
                            if (16 * pass + r < mine) *reinterpret_cast<uint4*>(dst + (size_t)(16 * pass + r) * (4 * D_V)) = v;
                        }
                        __syncwarp();
                    }
                }
            }
            tc_fence_before();
        }
    } else if (warp < PP_S_WARP) {
        // =================================================================== rows into the stages, and the queries
        // K: a warp has the first and third, or the second and fourth, of four groups of two or three chunks; V: two chunks of 64 rows.  A group has
        // its barriers; the bytes of both CTAs' K go to the even one's.
        const bool is_k = warp < PP_V0;
        const int g = is_k ? warp - PP_K0 : warp - PP_V0, rows = p.copy_rows, half = 64 / rows;        // copies of 64 rows
        const int h = is_k ? (int)rank : g >> 1, i0 = h * half;   // which 64 rows of a block
        BlockWalk walk(p, piece);
        BlockPlaces w;
        uint32_t pieces = 0;
        bool ok = true;
        walk.look_up(p, row0, w);
        for (uint32_t it = 0; w.have; ++it) {
            // What can be done before the wait is; copies of less than 64 rows are handed from lane to lane after it.
            const uint32_t bytes = copies_of(w, i0, i0 + half) * (uint32_t)(rows * 128) + (is_k && w.first ? G_CHUNK : 0u);       // of a chunk
            const int e0 = __shfl_sync(0xffffffffu, w.page[0], i0 & 31), y0 = __shfl_sync(0xffffffffu, w.in[0], i0 & 31);
            if (is_k && w.first && pieces > 0) ok = mbar_wait_lean(bar(PB_QFREE), (pieces - 1) & 1u, abort_addr, WQ_QFREE);
#pragma unroll 1
            for (int n = g; n < 4 && ok; n += is_k ? 2 : 4) {
                const int c0 = is_k ? 2 * n : 4 * (int)rank + 2 * (g & 1), c1 = is_k && n == 3 ? PP_CHUNKS : c0 + 2;
                const uint32_t dst = is_k ? base + PPK_OFF + c0 * G_CHUNK : base + PPV_OFF + (4 * h + 2 * (g & 1)) * G_CHUNK;
                const uint32_t full = is_k ? barp(PB_KFULLP + n) : mapa_shared(bar(PB_VFULL + h), rank);
                if (it >= 1) ok = mbar_wait_lean(bar(is_k ? PB_KFREE + n : PB_VFREE + h), (it - 1) & 1u, abort_addr, is_k ? WQ_KFREE : WQ_VFREE);
                if (!ok) break;
                if (elect_one()) {
                    // Which rows are there: by the lane whose arrival hands it over.  (The slot's last readers, the softmax warps eight blocks
                    // ago, gave their score buffer back long before.)
                    if (is_k && n == 0) *reinterpret_cast<uint4*>(sm + PPY_OFF + 16 * (it & 7)) = make_uint4(w.valid[0], w.valid[1], w.valid[2], w.valid[3]);
                    mbar_arrive_expect_tx_remote(full, (uint32_t)(c1 - c0) * bytes);
                    if (half == 1 && e0 >= 0) {
#pragma unroll 1
                        for (int ch = c0; ch < c1; ++ch) tma_load_3d_pair(dst + (ch - c0) * G_CHUNK, &k_map, ch * 64, y0, e0, full);
                    }
                    if (is_k && w.first) {
#pragma unroll 1
                        for (int ch = c0; ch < c1; ++ch) tma_load_2d_pair(base + PPQ_OFF + ch * G_CHUNK, &q_map, ch * 64, w.q_row, full);
                    }
                }
                __syncwarp();
                if (half > 1)
                    each_copy(w, i0, i0 + half, [&](int i, int e, int y) {
#pragma unroll 1
                        for (int ch = c0; ch < c1; ++ch) tma_load_3d_pair(dst + (ch - c0) * G_CHUNK + (i - i0) * rows * 128, &k_map, ch * 64, y, e, full);
                    });
            }
            if (!ok) break;
            if (w.first) ++pieces;
            // The next block's places, and its rows asked into L2: what waits for a free stage should not wait for HBM as well.
            walk.look_up(p, row0, w);
            if (is_k && w.have)
                each_copy(w, i0, i0 + half, [&](int, int e, int y) {
#pragma unroll 1
                    for (int ch = g; ch < PP_CHUNKS; ch += 2) tma_prefetch_3d(&k_map, ch * 64, y, e);
                });
        }
    } else if (warp == PP_S_WARP) {
        // =================================================================== scores (even CTA)
        constexpr uint32_t idesc = instr_desc(F16 ? FMT_F16 : FMT_BF16, F16 ? FMT_F16 : FMT_BF16, false, false, 128, PP_TILE);
        const uint32_t q_lo = desc_lo(base + PPQ_OFF, 16), k_lo = desc_lo(base + PPK_OFF, 16);
        uint32_t it = 0;
        bool ok = rank == 0;
        while (ok && piece.next(p)) {
            for (int b = piece.b0; b < piece.b1 && ok; ++b, ++it) {
                const uint32_t st = it & 1;
                if (it >= 2) ok = mbar_wait_lean(bar(PB_SFREEP + st), ((it >> 1) - 1) & 1u, abort_addr, WQ_SFREE);
#pragma unroll 1
                for (int g = 0; g < 4 && ok; ++g) {
                    ok = mbar_wait_lean(bar(PB_KFULLP + g), it & 1u, abort_addr, WQ_KFULL);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t d = tmem + PPT_S + 64 * st;
#pragma unroll 1
                        for (int ch = 2 * g; ch < (g == 3 ? PP_CHUNKS : 2 * g + 2); ++ch) {
                            const uint32_t qa = q_lo + ((ch * G_CHUNK) >> 4), ka = k_lo + ((ch * G_CHUNK) >> 4);
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                mma_pair_f16(d, make_desc(qa + 2 * k, PP_DESC_HI), make_desc(ka + 2 * k, PP_DESC_HI), idesc, (ch | k) != 0);
                        }
                        commit_both(PB_KFREE + g);
                        if (g == 3) {
                            commit_both(PB_SREADY + st);
                            if (b + 1 == piece.b1) commit_both(PB_QFREE);
                        }
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp == PP_PV_WARP) {
        // =================================================================== P.V (odd CTA: its V has landed)
        constexpr uint32_t idesc = instr_desc(F16 ? FMT_F16 : FMT_BF16, F16 ? FMT_F16 : FMT_BF16, false, true, 128, 256);
        const uint32_t p_lo = desc_lo(base + PPP_OFF, 16), v_lo = desc_lo(base + PPV_OFF, G_CHUNK), v_peer = barp(PB_VPEERP);   // V: the next 64 dims lie a chunk further
        uint32_t it = 0;
        bool ok = true;
        while (ok && piece.next(p)) {
            for (int b = piece.b0; b < piece.b1 && ok; ++b, ++it) {
#pragma unroll 1
                for (int h = 0; h < 2 && ok; ++h) {
                    ok = mbar_wait_lean(bar(PB_VFULL + h), it & 1u, abort_addr, WQ_VFULL);
                    if (ok && rank == 0) ok = mbar_wait_lean(bar(PB_VPEERP + h), it & 1u, abort_addr, WQ_VPEER);
                    if (ok && rank == 0) ok = mbar_wait_lean(bar(PB_PREADYP + h), it & 1u, abort_addr, WQ_PREADY);
                    if (!ok) break;
                    if (rank != 0) {
                        if (lane == 0) mbar_arrive_remote(v_peer + 8 * h);
                        continue;
                    }
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                mma_pair_f16(tmem + PPT_O + 128 * n, make_desc(p_lo + ((h * G_CHUNK + k * 32) >> 4), PP_DESC_HI),
                                             make_desc(v_lo + (((4 * h + 2 * n) * G_CHUNK + k * 2048) >> 4), PP_DESC_HI), idesc,
                                             b != piece.b0 || h != 0 || k != 0);
                        }
                        commit_both(PB_VFREE + h);        // (of half 1: all products of the block)
                    }
                    __syncwarp();
                }
            }
        }
    }

    if (*abort_flag != 0) {        // a wait gave up: copies and MMAs may still be in flight; give them time to finish
        const long long t0 = clock64();
        while (clock64() - t0 < 200000) { }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();            // the partner may still arrive on this CTA's barriers until here
    if (tid == 0 && *abort_flag != 0 && p.status != nullptr) {
        atomicCAS(p.status, 0, *abort_flag);
        atomicAdd(p.status + 1, 1);
        p.status[2] = blockIdx.x;
    }
    if (warp == PP_S_WARP) { tc_fence_after(); tmem_dealloc_pair(tmem, 512); }
}

}  // namespace

int launch_attn_paged_pair(const PagedParams& p, bool f16, const CUtensorMap& q_map, const CUtensorMap& k_map, cudaStream_t stream) {
    static std::atomic<bool> attr_set[64];
    const auto kernel = f16 ? attn_paged_pair_kernel<true> : attn_paged_pair_kernel<false>;
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return set_error(SMLA_E_SHAPE, "attn_paged_pair_kernel: device ordinal %d not supported", dev);
    if (!attr_set[dev]) {
        for (const auto k : {attn_paged_pair_kernel<true>, attn_paged_pair_kernel<false>}) {
            const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PP_SMEM);
            if (e != cudaSuccess) return set_error((int)e, "attn_paged_pair_kernel: cannot reserve %u bytes of shared memory: %s", PP_SMEM, cudaGetErrorString(e));
        }
        attr_set[dev] = true;
    }
    launch_dependent(kernel, dim3(2 * p.num_parts, (p.rows + PP_TILE - 1) / PP_TILE), dim3(PP_THREADS), PP_SMEM, stream, p, q_map, k_map);
    return check_launch("attn_paged_pair_kernel");
}

}  // namespace smla
