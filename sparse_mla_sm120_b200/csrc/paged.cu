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
// Warps: 0-7 softmax and epilogue (16 query rows by half of the block's rows each); one that issues the score MMAs and one for P.V; and
// who brings the rows into two stages of 72 KB: four warps by TMA (16-bit rows), or eight through registers (packed rows: e4m3 x its scale
// is exact in bf16 where scales are powers of two, as the writers make them; four for even blocks, four for odd ones).  A stage is filled and freed in four groups of 128 dims, so that scores
// begin when a quarter of the rows is there, and the next rows come when P.V is through with a quarter.
// Every wait is bounded; a wait that gives up records a code in status[] and the CTA drains and exits.
//
// Which calls come here: up to 64 query rows per request, and packed rows; more query rows of 16-bit caches go to paged_pair.cu (64
// requests of up to 8192 rows, 128 heads: 149.6 us here with every row read by two CTAs, 114 to 118 there).
// What bounds it: with few query rows the products, whose operands of 64 rows make shared memory the limit (36 + 16 products of a block: 2300
// cycles for 16 query rows as for 64), of a block's 2700 to 3100; a call of a few blocks is a chain of latencies (entry, lengths, table, rows,
// four blocks, epilogue, merge: 13.8 us for 1000 rows).  Packed rows: the way through registers, about 5000 cycles for a warp's 16 rows.
// 48 requests of up to 4096 fp16 rows in pages of 16, two tokens of 16 heads: 44.5 us, 2.9 TB/s; 656-byte rows, 64 requests of up to 8192, 64
// heads: 102 us; 584-byte, 13 of up to 16384, 128 heads: 92.5 us.  Of a prompt's chunk under a causal mask all blocks are walked, also those that
// no query row of the CTA sees (256 tokens of 16 heads over 4096 rows: bf16 54 us, 656-byte 126).
// What the steps brought (the first version, rows by one warp and one stage of waiting: 52.5, 122.8, 104.7 us): rows by TMA from four warps and
// stages in quarters 49.1, 118.9, 94.0; rows asked into L2 ahead and a shorter epilogue 44.6, 116.8, 96.8; fewer registers spilled (a spilled
// register costs hundreds of cycles beside 220 KB of shared memory) and packed rows asked into L2 ahead 44.5, 101.9, 91.9;
// hidden rows judged by their values 44.5, 101.8, 92.6.  Measured and not
// kept: a packed row's values asked for as soon as those of the block before are in the stage (160, 110: the fence before a stage is handed over
// waits for the loads).
#include "paged_common.cuh"
#include "rows_map.cuh"

namespace smla {

namespace {

using namespace ptx;
using namespace attn;

constexpr int PG_ROWS = 64;                       // query rows of a CTA
constexpr int PG_SM_WARPS = 8, PG_SM_THREADS = PG_SM_WARPS * 32;
__host__ __device__ constexpr bool packed_rows(int layout) { return layout == SMLA_LAYOUT_V32 || layout == SMLA_LAYOUT_MODEL1; }
__host__ __device__ constexpr int load_warps(int layout) { return packed_rows(layout) ? 8 : 4; }
__host__ __device__ constexpr int paged_threads(int layout) { return packed_rows(layout) ? 640 : 448; }       // (packed: whole groups of four warps)
// registers of the packed layouts' instances, which the loading warps take from the others
constexpr int PG_REGS_LAUNCH = 96, PG_REGS_SOFTMAX = 96, PG_REGS_LOAD = 120, PG_REGS_MMA = 48;
static_assert(PG_REGS_SOFTMAX == PG_REGS_LAUNCH && PG_REGS_LOAD >= PG_REGS_LAUNCH && PG_REGS_MMA <= PG_REGS_LAUNCH, "who gives registers and who takes");
static_assert(PG_SM_WARPS * 32 * PG_REGS_SOFTMAX + 8 * 32 * PG_REGS_LOAD + 4 * 32 * PG_REGS_MMA <= 640 * PG_REGS_LAUNCH, "register budgets exceed what the CTA owns");

constexpr uint32_t G_STAGE = 9 * G_CHUNK;
constexpr uint32_t GQ_OFF = 0;
constexpr uint32_t GK_OFF = GQ_OFF + G_STAGE;
constexpr uint32_t GP_OFF = GK_OFF + 2 * G_STAGE;             // weights [64 query rows][64 rows] 16-bit
constexpr uint32_t GV_OFF = GP_OFF + G_CHUNK;                 // validity: a bit per row, [2 stages] 64 bits
constexpr uint32_t GA_OFF = GV_OFF + 16;                      // [64] fp32: rescale factors, then 1 / denominator
constexpr uint32_t GX_OFF = GA_OFF + PG_ROWS * 4;             // [2][64] fp32: maxima, then sums, of the two halves of a block's rows
constexpr uint32_t GW_OFF = GX_OFF + 2 * PG_ROWS * 4;         // schedule
constexpr uint32_t GB_OFF = GW_OFF + 24 * 8;
// KFULL, KFREE: [2 stages][4 groups of dims]
constexpr int GB_KFULL = 0, GB_KFREE = 8, GB_SREADY = 16, GB_SFREE = 18, GB_PREADY = 20, GB_PVDONE = 21, GB_QFREE = 22, GB_N = 23;
constexpr uint32_t GMISC_OFF = GB_OFF + GB_N * 8;
constexpr uint32_t G_SMEM = GMISC_OFF + 16 + 1024;
static_assert(G_SMEM <= 227 * 1024, "shared memory budget");
static_assert(GB_OFF % 8 == 0 && GA_OFF % 16 == 0 && GW_OFF % 8 == 0, "alignment");

constexpr uint32_t GT_O = 0, GT_S = 256;          // tensor memory: dims block b of O^T at 64 b, the two score buffers at 256 and 320
constexpr uint32_t G_DESC_HI = desc_hi(1024, (uint32_t)SWIZZLE_128B);

enum { WP_KFULL = 61, WP_KFREE = 62, WP_SREADY = 63, WP_PREADY = 64, WP_PVDONE = 65, WP_QFREE = 66, WP_SFREE = 67 };

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

template <int LAYOUT> __global__ void __launch_bounds__(paged_threads(LAYOUT), 1)
attn_paged_kernel(const PagedParams p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map) {
    constexpr bool F16 = LAYOUT == SMLA_LAYOUT_F16, PACKED = packed_rows(LAYOUT);
    constexpr int CHUNKS = LAYOUT == SMLA_LAYOUT_MODEL1 ? 8 : 9;
    constexpr int LD0 = PG_SM_WARPS, S_WARP = LD0 + load_warps(LAYOUT), PV_WARP = S_WARP + 1, WARPS = paged_threads(LAYOUT) / 32;
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
        for (int i = 0; i < 8; ++i) {
            mbar_init(bar(GB_KFULL + i), PACKED ? 4 : 1);
            mbar_init(bar(GB_KFREE + i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(GB_SREADY + i), 1);
            mbar_init(bar(GB_SFREE + i), PG_SM_WARPS);
        }
        mbar_init(bar(GB_PREADY), PG_SM_WARPS);
        mbar_init(bar(GB_PVDONE), 1);
        mbar_init(bar(GB_QFREE), 1);
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == S_WARP) { tmem_alloc(base + GMISC_OFF, 512); tmem_relinquish(); }
    grid_dep_wait();
    grid_dep_launch();

    Pieces<64> piece = partition_of<64>(p, part, reinterpret_cast<long long*>(sm + GW_OFF), WARPS);
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + GMISC_OFF);
    if (PACKED) {
        if (warp >= S_WARP) setmaxnreg_dec<PG_REGS_MMA>();
        else if (warp >= LD0) setmaxnreg_inc<PG_REGS_LOAD>();
    }

    if (warp < PG_SM_WARPS) {
        // =================================================================== softmax + epilogue
        // The thread's query rows ra and rb, and of a block's rows [32 half, +32) the columns 8 i + 2 (lane % 4) + {0, 1}.
        const int quarter = warp & 3, half = warp >> 2, quad = lane & 3;
        const int ra = 16 * quarter + (lane >> 2), rb = ra + 8;
        const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
        const float c = p.sm_scale * LOG2E;
        float* factor = reinterpret_cast<float*>(sm + GA_OFF);
        float* other = reinterpret_cast<float*>(sm + GX_OFF);
        const bool busy = live > 32 * half;                       // the half has columns of O^T
        uint32_t it = 0;
        bool dead = false, stop = false;
        while (!stop && piece.next(p)) {
            const bool whole = piece.whole();
            if (row0 == 0 && tid == 0 && piece.b0 == 0) {
                piece.write_span(p, part, reinterpret_cast<long long*>(sm + GW_OFF)[20]);
            }
            const int see_a = paged_sees(p, piece.len, row0 + ra), see_b = paged_sees(p, piece.len, row0 + rb), see_least = paged_sees(p, piece.len, row0);
            float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;
            for (int b = piece.b0; b < piece.b1; ++b, ++it) {
                const uint32_t st = it & 1;
                if (!dead) dead = !mbar_wait_lean(bar(GB_SREADY + st), (it >> 1) & 1u, abort_addr, WP_SREADY);
                uint32_t sv[16];
                float mx_a = -INFINITY, mx_b = -INFINITY;
                const int pos0 = b * 64;
                unsigned long long valid = ~0ull;
                if (!dead) {
                    tc_fence_after();
                    tmem_ld_16x256b_x4(lane_addr + GT_S + 64 * st + 32 * half, sv);
                    valid = *reinterpret_cast<volatile unsigned long long*>(sm + GV_OFF + 8 * st);
                    tmem_wait_ld();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(GB_SFREE + st));
                    if (valid == ~0ull && pos0 <= see_least - 64) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) sv[i] = __float_as_uint(__uint_as_float(sv[i]) * c);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int at = 32 * half + 8 * (i >> 2) + 2 * quad + (i & 1);
                            const bool seen = ((valid >> at) & 1) && pos0 + at < ((i & 2) ? see_b : see_a);
                            sv[i] = __float_as_uint(seen ? __uint_as_float(sv[i]) * c : -INFINITY);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        mx_a = fmaxf(mx_a, fmaxf(__uint_as_float(sv[i]), __uint_as_float(sv[i + 1])));
                        mx_b = fmaxf(mx_b, fmaxf(__uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3])));
                    }
#pragma unroll
                    for (int o = 1; o <= 2; o <<= 1) {
                        mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, o));
                        mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, o));
                    }
                }
                if (quad == 0) { other[half * PG_ROWS + ra] = mx_a; other[half * PG_ROWS + rb] = mx_b; }
                const bool grow = mx_a > m_a + PG_TAU || mx_b > m_b + PG_TAU;                // false while a row has seen nothing
                if (named_bar_or(1, PG_SM_THREADS, grow || dead || *abort_flag != 0)) {
                    // rare: a maximum grows, or the CTA gives up
                    const float all_a = fmaxf(other[ra], other[PG_ROWS + ra]), all_b = fmaxf(other[rb], other[PG_ROWS + rb]);
                    float al_a = 1.f, al_b = 1.f;
                    if (all_a > m_a + PG_TAU) { al_a = ex2(m_a - all_a); m_a = all_a; l_a *= al_a; }
                    if (all_b > m_b + PG_TAU) { al_b = ex2(m_b - all_b); m_b = all_b; l_b *= al_b; }
                    if (quad == 0 && half == 0) { factor[ra] = al_a; factor[rb] = al_b; }
                    if (b > piece.b0 && !dead) dead = !mbar_wait_lean(bar(GB_PVDONE), (it - 1) & 1u, abort_addr, WP_PVDONE);
                    if (named_bar_or(1, PG_SM_THREADS, dead || *abort_flag != 0)) { stop = true; break; }
                    if (b > piece.b0 && busy) {
                        tc_fence_after();
#pragma unroll 1
                        for (int d = 0; d < 8; ++d) {
                            const uint32_t at = lane_addr + GT_O + 64 * (d >> 1) + 32 * half + 16 * (d & 1);
                            uint32_t o[16];
                            tmem_ld16(at, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor[32 * half + 16 * (d & 1) + i]);
                            tmem_st16(at, o);
                        }
                        tmem_wait_st();
                    }
                    named_bar_sync(1, PG_SM_THREADS);             // the factors and maxima have been read
                }
                const float ma = m_a == -INFINITY ? 0.f : m_a, mb = m_b == -INFINITY ? 0.f : m_b;
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a0 = ex2(__uint_as_float(sv[4 * i]) - ma), a1 = ex2(__uint_as_float(sv[4 * i + 1]) - ma);
                    const float b0 = ex2(__uint_as_float(sv[4 * i + 2]) - mb), b1 = ex2(__uint_as_float(sv[4 * i + 3]) - mb);
                    l_a += a0 + a1;
                    l_b += b0 + b1;
                    w[2 * i] = pack_weights<F16>(a0, a1);
                    w[2 * i + 1] = pack_weights<F16>(b0, b1);
                }
                // the weights of the block before have been read
                if (it > 0 && !dead) dead = !mbar_wait_lean(bar(GB_PVDONE), (it - 1) & 1u, abort_addr, WP_PVDONE);
                if ((valid != ~0ull || pos0 > see_least - 64) && !dead) {
                    // Rows that are not there, and values that are no numbers in rows hidden from some query, would reach queries through
                    // 0 x V: they are taken out of the stage, whose scores are done.  (By the rows' values, not by scores, which a query that is
                    // no number spoils too.  A query that sees such a row has a weight that is no number.)
#pragma unroll 1
                    for (int g = 0; g < (PACKED ? 1 : 4) && !dead; ++g)       // over since the scores are there: what copies wrote is read here
                        dead = !mbar_wait_lean(bar(GB_KFULL + 4 * st + g), (it >> 1) & 1u, abort_addr, WP_KFULL);
#pragma unroll 1
                    for (int i = tid; i < 64 * (D_V / 8); i += PG_SM_THREADS) {
                        const int r = (i >> 3) & 63;
                        uint4* at = reinterpret_cast<uint4*>(sm + GK_OFF + st * G_STAGE + (i >> 9) * G_CHUNK + r * 128 + (i & 7) * 16);
                        if (!((valid >> r) & 1)) *at = make_uint4(0, 0, 0, 0);
                        else if (pos0 + r >= see_least) *at = numbers_only<F16>(*at);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    *reinterpret_cast<uint32_t*>(sm + GP_OFF + gswz((uint32_t)ra, (uint32_t)(4 * half + i)) + 4 * quad) = w[2 * i];
                    *reinterpret_cast<uint32_t*>(sm + GP_OFF + gswz((uint32_t)rb, (uint32_t)(4 * half + i)) + 4 * quad) = w[2 * i + 1];
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
            if (quad == 0) { other[half * PG_ROWS + ra] = l_a; other[half * PG_ROWS + rb] = l_b; }
            if (named_bar_or(1, PG_SM_THREADS, dead || *abort_flag != 0)) { stop = true; break; }
            const size_t rec = whole ? (size_t)piece.req : (size_t)(2 * part + (piece.b0 == 0 ? 1 : 0));
            if (half == 0 && quad < 2) {                          // one lane for each of the quad's rows
                const int r = quad == 0 ? ra : rb;
                const float l = other[r] + other[PG_ROWS + r], m = quad == 0 ? m_a : m_b;
                float lse = l == 0.f ? (whole ? NEG_BIG : NO_RECORD) : log2f(l) + m, denom = l;
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
            named_bar_sync(1, PG_SM_THREADS);
            // 16 query rows at a time: their factors, then their 128 dims of the warp's lanes from all four accumulators
#pragma unroll 1
            for (int r0 = 32 * half; r0 < min(live, 32 * half + 32); r0 += 16) {
                float f[16];
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(factor + r0 + i);
                    f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
                }
                const size_t at = (rec * p.rows + row0 + r0) * D_V + 32 * quarter + lane;
                const int left = live - r0;
                auto store = [&](auto* dst, auto cvt) {
#pragma unroll 1
                    for (int d = 0; d < 4; ++d) {
                        uint32_t o[16];
                        if (piece.b1 > piece.b0) tmem_ld16(lane_addr + GT_O + 64 * d + r0, o);
                        tmem_wait_ld();
                        if (left >= 16) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) dst[128 * d + i * D_V] = cvt(f[i] == 0.f ? 0.f : __uint_as_float(o[i]) * f[i]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (i < left) dst[128 * d + i * D_V] = cvt(f[i] == 0.f ? 0.f : __uint_as_float(o[i]) * f[i]);
                        }
                    }
                };
                if (whole) store(static_cast<uint16_t*>(p.out) + at, [](float v) { return out_bits<F16>(v); });
                else store(p.o_part + at, [](float v) { return v; });
            }
            tc_fence_before();
            named_bar_sync(1, PG_SM_THREADS);                     // the factors have been read
        }
    } else if (warp < S_WARP) {
        // =================================================================== rows into the stages, and the queries
        uint32_t it = 0, pieces = 0;
        bool ok = true;
        if constexpr (!PACKED) {
            // A warp per group of dims: a copy takes its warp about 130 cycles to issue, all of them from one warp 3900 cycles a block.
            const int rows = p.copy_rows, copies = 64 / rows;     // rows of a copy, copies of a block (and chunk): lane i sees to i and i + 32
            const int g = warp - LD0, c0 = 2 * g, c1 = g == 3 ? CHUNKS : c0 + 2;
            // Where a block's rows lie, and which of them are there; looked up two blocks ahead and asked into L2 then: what waits for a
            // free stage should not wait for HBM as well.
            struct Places {
                int page[2], in[2], q_row;
                unsigned v_lo, v_hi;
                uint32_t bytes;                                   // of a chunk
                bool have, first;                                 // there is such a block; it is the first of its piece
            };
            int b = -1;
            bool more = piece.next(p);
            auto look_up = [&](Places& w) {                       // the next block in line
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
                unsigned long long valid = 0ull;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int i = lane + 32 * u, pos = b * 64 + i * rows;
                    w.page[u] = -1;
                    w.in[u] = 0;
                    if (i < copies && pos < piece.len) {
                        const int j = pos / p.page_block_size, e = ld_in(p.table + (int64_t)piece.req * p.table_stride + j);
                        if (e >= 0 && e < p.num_pages) {
                            w.page[u] = e;
                            w.in[u] = pos - j * p.page_block_size;
                            const int k = min(piece.len - pos, rows);
                            valid |= (k == 64 ? ~0ull : (1ull << k) - 1ull) << (i * rows);
                        }
                    }
                }
                w.v_lo = __reduce_or_sync(0xffffffffu, (unsigned)valid);
                w.v_hi = __reduce_or_sync(0xffffffffu, (unsigned)(valid >> 32));
                w.bytes = (uint32_t)(__popc(__ballot_sync(0xffffffffu, w.page[0] >= 0)) + __popc(__ballot_sync(0xffffffffu, w.page[1] >= 0))) * rows * 128u;
                if (++b == piece.b1) {
                    more = piece.next(p);
                    b = -1;
                }
            };
            auto copy = [&](const Places& w, auto&& one) {        // one(copy's number, its page, its first row), under elect_one, with operands that are the same in all lanes
#pragma unroll 1
                for (int i = 0; i < copies; ++i) {
                    const int e = __shfl_sync(0xffffffffu, i < 32 ? w.page[0] : w.page[1], i & 31), y = __shfl_sync(0xffffffffu, i < 32 ? w.in[0] : w.in[1], i & 31);
                    if (e >= 0 && elect_one()) one(i, e, y);
                }
                __syncwarp();
            };
            Places w0, w1;
            look_up(w0);
            look_up(w1);
            for (; w0.have && ok; ++it) {
                const uint32_t st = it & 1, full = bar(GB_KFULL + 4 * st + g);
                if (it >= 2) ok = mbar_wait_lean(bar(GB_KFREE + 4 * st + g), ((it >> 1) - 1) & 1u, abort_addr, WP_KFREE);
                if (ok && w0.first && pieces > 0) ok = mbar_wait_lean(bar(GB_QFREE), (pieces - 1) & 1u, abort_addr, WP_QFREE);
                if (!ok) break;
                if (elect_one()) {
                    // (by the lane whose arrival hands them over)
                    if (g == 0) *reinterpret_cast<volatile unsigned long long*>(sm + GV_OFF + 8 * st) = ((unsigned long long)w0.v_hi << 32) | w0.v_lo;
                    mbar_arrive_expect_tx(full, (uint32_t)(c1 - c0) * (w0.bytes + (w0.first ? G_CHUNK : 0u)));
                    if (w0.first)
                        for (int ch = c0; ch < c1; ++ch) tma_load_2d(base + GQ_OFF + ch * G_CHUNK, &q_map, ch * 64, w0.q_row, full);
                }
                const uint32_t dst = base + GK_OFF + st * G_STAGE;
                copy(w0, [&](int i, int e, int y) {
                    for (int ch = c0; ch < c1; ++ch) tma_load_3d(dst + ch * G_CHUNK + i * rows * 128, &k_map, ch * 64, y, e, full);
                });
                if (w0.first) ++pieces;
                w0 = w1;
                look_up(w1);
                if (w1.have)
                    copy(w1, [&](int, int e, int y) {
                        for (int ch = c0; ch < c1; ++ch) tma_prefetch_3d(&k_map, ch * 64, y, e);
                    });
            }
        } else {
            const int stage = (warp - LD0) >> 2, gw = (warp - LD0) & 3;
            const uint32_t kst = GK_OFF + stage * G_STAGE;
            constexpr int NOPE = LAYOUT == SMLA_LAYOUT_V32 ? D_NOPE : 448;
            constexpr int ROPE_AT = LAYOUT == SMLA_LAYOUT_V32 ? ROPE_OFF : 448;
            while (ok && piece.next(p)) {
                if (piece.b1 == piece.b0) continue;
                const int32_t* table = p.table + (int64_t)piece.req * p.table_stride;
                // lane i: where row i % 16 of the warp's rows of a block lies (0: no entry)
                auto look_up = [&](int b, uint2& scales) {
                    scales = make_uint2(0u, 0u);
                    const int pos = b * 64 + 16 * gw + (lane & 15);
                    if (pos >= piece.len) return 0ull;
                    const int j = pos / p.page_block_size, page = ld_in(table + j), in = pos - j * p.page_block_size;
                    if (page < 0 || page >= p.num_pages) return 0ull;
                    const uint8_t* mine = p.cache + (int64_t)page * p.page_stride;
                    if (LAYOUT == SMLA_LAYOUT_MODEL1)
                        scales = ld_in(reinterpret_cast<const uint2*>(mine + (int64_t)p.page_block_size * SMLA_M1_DATA_BYTES + (int64_t)in * 8));
                    return reinterpret_cast<unsigned long long>(mine + (int64_t)in * (LAYOUT == SMLA_LAYOUT_V32 ? ROW_BYTES : SMLA_M1_DATA_BYTES));
                };
                unsigned long long at = 0ull, next_at = 0ull;
                uint2 sc8 = make_uint2(0u, 0u), next_sc8 = sc8;
                bool known = false;
                for (int b = piece.b0; b < piece.b1 && ok; ++b, ++it) {
                    if ((it & 1) != (uint32_t)stage) continue;
                    if (known) { at = next_at; sc8 = next_sc8; }
                    else at = look_up(b, sc8);
                    const unsigned bits = __ballot_sync(0xffffffffu, at != 0ull) & 0xffffu;
                    uint4 nope[16], rope[4];
                    float scale[2] = {0.f, 0.f};                  // of row lane / 4 (+ 8), block lane % 4 of 128 dims
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint8_t* src = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, at, i));
                        nope[i] = make_uint4(0, 0, 0, 0);
                        if (src != nullptr && lane < NOPE / 16) nope[i] = ld_in_once(reinterpret_cast<const uint4*>(src) + lane);
                    }
                    if (LAYOUT == SMLA_LAYOUT_V32) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const uint8_t* src = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, at, (lane >> 2) + 8 * u));
                            if (src != nullptr) scale[u] = ld_in(reinterpret_cast<const float*>(src + SCALE_OFF) + (lane & 3));
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint8_t* src = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, at, 4 * u + (lane >> 3)));
                        rope[u] = make_uint4(0, 0, 0, 0);
                        if (src != nullptr) rope[u] = ld_in_once(reinterpret_cast<const uint4*>(src + ROPE_AT) + (lane & 7));
                    }
                    // The warp's next rows, asked into L2 while these are on their way and turned into the stage.
                    known = b + 2 < piece.b1;
                    if (known) {
                        next_at = look_up(b + 2, next_sc8);
                        if (next_at != 0ull) {
#pragma unroll
                            for (int i = 0; i < 3; ++i) prefetch_l2(reinterpret_cast<const uint8_t*>(next_at) + min(128 * (2 * i + (lane >> 4)), ROPE_AT + 127));
                        }
                    }
                    if (it >= 2) ok = mbar_wait_lean(bar(GB_KFREE + 4 * stage + 3), ((it >> 1) - 1) & 1u, abort_addr, WP_KFREE);
                    if (!ok) break;
                    const uint32_t full = bar(GB_KFULL + 4 * stage);
                    const bool queries = b == piece.b0 && gw == 0;       // the piece's queries come with its first block
                    if (queries) {
                        if (pieces > 0) ok = mbar_wait_lean(bar(GB_QFREE), (pieces - 1) & 1u, abort_addr, WP_QFREE);
                        if (!ok) break;
                        if (elect_one()) {
                            mbar_expect_tx(full, CHUNKS * G_CHUNK);
                            for (int ch = 0; ch < CHUNKS; ++ch) tma_load_2d(base + GQ_OFF + ch * G_CHUNK, &q_map, ch * 64, piece.req * p.rows + row0, full);
                        }
                        __syncwarp();
                    }
                    const uint32_t chunk = kst + (lane >> 2) * G_CHUNK;
                    const bool swap = (lane & 4) != 0;           // neighbouring chunks store their two pieces in opposite order: no bank conflicts
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint32_t r = (uint32_t)(16 * gw + i), pc = 2u * (lane & 3);
                        float f;
                        if (LAYOUT == SMLA_LAYOUT_V32) {
                            f = __shfl_sync(0xffffffffu, scale[i >> 3], 4 * (i & 7) + (lane >> 3));
                        } else {
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
                    if (lane == 0) *reinterpret_cast<volatile uint16_t*>(sm + GV_OFF + 8 * stage + 2 * gw) = (uint16_t)bits;
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full);
                }
                ++pieces;
            }
        }
    } else if (warp == S_WARP) {
        // =================================================================== scores
        const uint32_t idesc = instr_desc(F16 ? FMT_F16 : FMT_BF16, F16 ? FMT_F16 : FMT_BF16, false, false, 64, 64);
        const uint32_t q_lo = desc_lo(base + GQ_OFF, 16), k_lo = desc_lo(base + GK_OFF, 16);
        uint32_t it = 0;
        bool ok = true;
        while (ok && piece.next(p)) {
            for (int b = piece.b0; b < piece.b1 && ok; ++b, ++it) {
                const uint32_t st = it & 1;
                if (it >= 2) ok = mbar_wait_lean(bar(GB_SFREE + st), ((it >> 1) - 1) & 1u, abort_addr, WP_SFREE);
#pragma unroll 1
                for (int g = 0; g < 4 && ok; ++g) {
                    if (!PACKED || g == 0) ok = mbar_wait_lean(bar(GB_KFULL + 4 * st + g), (it >> 1) & 1u, abort_addr, WP_KFULL);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t qa = q_lo + ((2 * g * G_CHUNK) >> 4), ka = k_lo + ((st * G_STAGE + 2 * g * G_CHUNK) >> 4), d = tmem + GT_S + 64 * st;
                        mma_f16(d, make_desc(qa, G_DESC_HI), make_desc(ka, G_DESC_HI), idesc, g != 0);
#pragma unroll
                        for (int k = 1; k < 8; ++k)
                            mma_f16(d, make_desc(qa + (((k >> 2) * G_CHUNK + (k & 3) * 32) >> 4), G_DESC_HI),
                                    make_desc(ka + (((k >> 2) * G_CHUNK + (k & 3) * 32) >> 4), G_DESC_HI), idesc, true);
                        if (CHUNKS == 9 && g == 3) {
#pragma unroll
                            for (int k = 8; k < 12; ++k)
                                mma_f16(d, make_desc(qa + (((k >> 2) * G_CHUNK + (k & 3) * 32) >> 4), G_DESC_HI),
                                        make_desc(ka + (((k >> 2) * G_CHUNK + (k & 3) * 32) >> 4), G_DESC_HI), idesc, true);
                        }
                        if (g == 3) {
                            tc_commit(bar(GB_SREADY + st));
                            if (b + 1 == piece.b1) tc_commit(bar(GB_QFREE));
                        }
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp == PV_WARP) {
        // =================================================================== P.V
        const uint32_t idesc = instr_desc(F16 ? FMT_F16 : FMT_BF16, F16 ? FMT_F16 : FMT_BF16, true, false, 128, (uint32_t)((live + 15) & ~15));
        const uint32_t v_lo = desc_lo(base + GK_OFF, G_CHUNK), p_lo = desc_lo(base + GP_OFF, 16);      // V MN-major: the next 64 dims lie a chunk further
        uint32_t it = 0;
        bool ok = true;
        while (ok && piece.next(p)) {
            for (int b = piece.b0; b < piece.b1 && ok; ++b, ++it) {
                const uint32_t st = it & 1;
                ok = mbar_wait_lean(bar(GB_PREADY), it & 1u, abort_addr, WP_PREADY);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t va = v_lo + ((st * G_STAGE) >> 4);
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_f16(tmem + GT_O + 64 * d, make_desc(va + ((2 * d * G_CHUNK + k * 2048) >> 4), G_DESC_HI),
                                    make_desc(p_lo + ((k * 32) >> 4), G_DESC_HI), idesc, k != 0 || b != piece.b0);
                        tc_commit(bar(GB_KFREE + 4 * st + d));
                    }
                    tc_commit(bar(GB_PVDONE));
                }
                __syncwarp();
            }
        }
    }

    if (*abort_flag != 0) {        // a wait gave up: copies and MMAs may still be in flight; give them time to finish
        const long long t0 = clock64();
        while (clock64() - t0 < 200000) { }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *abort_flag != 0 && p.status != nullptr) {
        atomicCAS(p.status, 0, *abort_flag);
        atomicAdd(p.status + 1, 1);
        p.status[2] = blockIdx.x;
    }
    if (warp == S_WARP) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

// Joins what a request's partitions left, a query row by one warp or, where requests lie in many partitions, by four or eight: warp w sums records
// w, w + W, ..., four of them asked for at a time.  It is a chain of latencies (one request of 131072 rows in 74 partitions: 64 us with one warp
// per row and a record at a time, 11 with four and four records, 9 with eight), unless there are many rows: then more rows at a time hide it
// (64 requests of 128 heads in 74 partitions: 25 us with four warps per row, 11 with one).  Requests within one partition are done.  The order of the sums is fixed.
constexpr int PC_ROWS = 4, PC_AHEAD = 4;            // rows of a block where a warp takes one
__host__ __device__ constexpr int combine_warps(int w) { return w > 1 ? w : PC_ROWS; }
template <bool F16, int W> __global__ void __launch_bounds__(combine_warps(W) * 32) paged_combine_kernel(const PagedParams p) {
    __shared__ float4 sums[W > 1 ? W - 1 : 1][D_V / 4];
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, warp = W > 1 ? threadIdx.x >> 5 : 0;
    const int64_t id = W > 1 ? blockIdx.x : (int64_t)blockIdx.x * PC_ROWS + (threadIdx.x >> 5);
    if (id >= (int64_t)p.batch * p.rows) return;
    const int req = (int)(id / p.rows), row = (int)(id - (int64_t)req * p.rows);
    const uint2 span = ld_in(reinterpret_cast<const uint2*>(p.spans + req));
    const int c0 = (int)span.x, n = span_parts(c0, (int)span.y, p.num_parts);
    if (n <= 1) return;
    auto record = [&](int s) { return (size_t)(s == 0 ? 2 * c0 + 1 : 2 * (c0 + s)) * p.rows + row; };
    float4 v[PC_AHEAD][4];
    auto load = [&](int s0) {
#pragma unroll
        for (int u = 0; u < PC_AHEAD; ++u)
            if (s0 + W * u < n) {
                const float4* src = reinterpret_cast<const float4*>(p.o_part + record(s0 + W * u) * D_V) + lane;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[u][i] = ld_in_once(src + 32 * i);
            }
    };
    load(warp);
    float mx = NO_RECORD, sum = 0.f;
    for (int s = lane; s < n; s += 32) mx = fmaxf(mx, ld_in(p.lse_part + record(s)));
    mx = warp_max(mx);
    for (int s = lane; s < n; s += 32) {
        const float x = ld_in(p.lse_part + record(s));
        sum += x == NO_RECORD ? 0.f : exp2f(x - mx);
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
    for (int s0 = warp; s0 < n; s0 += W * PC_AHEAD) {
        if (s0 > warp) load(s0);
#pragma unroll
        for (int u = 0; u < PC_AHEAD; ++u) {
            const int s = s0 + W * u;
            if (s >= n) break;
            const float x = ld_in(p.lse_part + record(s)), w = x == NO_RECORD ? 0.f : exp2f(x - mx) * inv;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[i].x += w * v[u][i].x; acc[i].y += w * v[u][i].y; acc[i].z += w * v[u][i].z; acc[i].w += w * v[u][i].w;
            }
        }
    }
    if constexpr (W > 1) {
        if (warp > 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[warp - 1][32 * i + lane] = acc[i];
        }
        __syncthreads();
        if (warp > 0) return;
#pragma unroll
        for (int w = 0; w < W - 1; ++w) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 x = sums[w][32 * i + lane];
                acc[i].x += x.x; acc[i].y += x.y; acc[i].z += x.z; acc[i].w += x.w;
            }
        }
    }
    if (lane == 0) p.lse[id] = lse;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint2 r = make_uint2(pack_weights<F16>(acc[i].x, acc[i].y), pack_weights<F16>(acc[i].z, acc[i].w));
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + (size_t)id * D_V + i * 128 + lane * 4) = r;
    }
}

}  // namespace

bool paged_on_pairs(int rows, int layout) { return rows > PG_ROWS && !packed_rows(layout); }

int paged_parts(int batch, int rows, int pages_per_request, int page_block_size, int num_parts, bool pairs) {
    if (num_parts > 0) return num_parts;
    const int sms = smla_num_sms();
    if (sms < 1) return 0;
    const int unit = pairs ? 2 * PG_ROWS : PG_ROWS;               // query rows, and cache rows of a block
    const int groups = (rows + unit - 1) / unit, room = pairs ? sms / 2 : sms, most = room / groups > 0 ? room / groups : 1;
    const long long blocks = ((long long)pages_per_request * page_block_size + unit - 1) / unit;
    const long long worth = (batch * (blocks + PG_START) + PG_START - 1) / PG_START;
    return worth < most ? (int)(worth > 0 ? worth : 1) : most;
}

int launch_attn_paged(PagedParams p, int layout, cudaStream_t stream) {
    typedef void (*Kernel)(const PagedParams, const CUtensorMap, const CUtensorMap);
    static std::atomic<bool> attr_set[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return set_error(SMLA_E_SHAPE, "attn_paged_kernel: device ordinal %d not supported", dev);
    if (!attr_set[dev]) {
        const Kernel kernels[4] = {attn_paged_kernel<SMLA_LAYOUT_V32>, attn_paged_kernel<SMLA_LAYOUT_MODEL1>, attn_paged_kernel<SMLA_LAYOUT_BF16>,
                                   attn_paged_kernel<SMLA_LAYOUT_F16>};
        for (int i = 0; i < 4; ++i) {
            cudaFuncAttributes fa;
            if (i < 2 && (cudaFuncGetAttributes(&fa, kernels[i]) != cudaSuccess || fa.numRegs != PG_REGS_LAUNCH))
                return set_error(SMLA_E_DEVICE, "attn_paged_kernel: compiled with %d registers per thread, the warpgroup budgets assume %d", fa.numRegs, PG_REGS_LAUNCH);
            const cudaError_t e = cudaFuncSetAttribute(kernels[i], cudaFuncAttributeMaxDynamicSharedMemorySize, (int)G_SMEM);
            if (e != cudaSuccess) return set_error((int)e, "attn_paged_kernel: cannot reserve %u bytes of shared memory: %s", G_SMEM, cudaGetErrorString(e));
        }
        attr_set[dev] = true;
    }
    CUtensorMap q_map{}, k_map{};
    const bool packed = packed_rows(layout), f16 = layout == SMLA_LAYOUT_F16;
    const CUtensorMapDataType type = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const uint64_t d = layout == SMLA_LAYOUT_MODEL1 ? SMLA_M1_D_QK : D_QK;
    const uint64_t q_dims[2] = {d, (uint64_t)p.batch * p.rows}, q_strides[1] = {2 * d};
    const uint32_t q_box[2] = {64, PG_ROWS};
    if (int e = encode_map(&q_map, type, 2, p.q, q_dims, q_strides, q_box, CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) return e;
    p.copy_rows = 64;                              // the largest power of two that divides pages and blocks
    while (p.page_block_size % p.copy_rows != 0) p.copy_rows >>= 1;
    if (!packed && p.num_pages > 0) {
        const uint64_t k_dims[3] = {D_QK, (uint64_t)p.page_block_size, (uint64_t)p.num_pages}, k_strides[2] = {2 * D_QK, (uint64_t)p.page_stride};
        const uint32_t k_box[3] = {64, (uint32_t)p.copy_rows, 1};
        if (int e = encode_map(&k_map, type, 3, p.cache, k_dims, k_strides, k_box, CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) return e;
    }
    const bool pairs = paged_on_pairs(p.rows, layout);
    if (pairs) {
        if (int e = launch_attn_paged_pair(p, f16, q_map, k_map, stream)) return e;
    }
    const Kernel kernel = layout == SMLA_LAYOUT_V32      ? attn_paged_kernel<SMLA_LAYOUT_V32>
                          : layout == SMLA_LAYOUT_MODEL1 ? attn_paged_kernel<SMLA_LAYOUT_MODEL1>
                          : layout == SMLA_LAYOUT_BF16   ? attn_paged_kernel<SMLA_LAYOUT_BF16>
                                                         : attn_paged_kernel<SMLA_LAYOUT_F16>;
    if (!pairs) {
        launch_dependent(kernel, dim3(p.num_parts, (p.rows + PG_ROWS - 1) / PG_ROWS), dim3(paged_threads(layout)), G_SMEM, stream, p, q_map, k_map);
        if (int e = check_launch("attn_paged_kernel")) return e;
    }
    if (p.num_parts == 1) return 0;                // every request is whole
    const unsigned rows = (unsigned)p.batch * (unsigned)p.rows;
    typedef void (*Combine)(const PagedParams);
    const int warps = p.num_parts >= 16 * (int64_t)p.batch ? 8 : p.num_parts >= 4 * (int64_t)p.batch ? 4 : 1;       // per row
    const Combine combine = warps == 8   ? (f16 ? paged_combine_kernel<true, 8> : paged_combine_kernel<false, 8>)
                            : warps == 4 ? (f16 ? paged_combine_kernel<true, 4> : paged_combine_kernel<false, 4>)
                                         : (f16 ? paged_combine_kernel<true, 1> : paged_combine_kernel<false, 1>);
    launch_dependent(combine, dim3(warps > 1 ? rows : (rows + PC_ROWS - 1) / PC_ROWS), dim3(combine_warps(warps) * 32), 0, stream, p);
    return check_launch("paged_combine_kernel");
}

}  // namespace smla
