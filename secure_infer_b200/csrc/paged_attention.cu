// paged_attention.cu -- attention of a chunk of new tokens over the paged KV
// cache, in one pass with the running maximum and sum of a softmax:
//
//   x_j = scale log2(e) q.k_j,  m' = max(m, x_j),  p_j = 2^(x_j - m'),
//   l' = l 2^(m - m') + sum p_j,  o' = o 2^(m - m') + sum p_j v_j,  out = o / l.
//
// (m, l, o) over two sets of keys join by the same rule, which is what splits a
// long context over CTAs.
#include "paged.cuh"
#include "gcm_kernels.cuh"

#include <atomic>
#include <mutex>

namespace sib {
namespace paged {
namespace {

// Workspace: the status word, counters, cuts, then partial results.
constexpr int kMaxGrid = 256;   // CTAs; a device with fewer SMs has as many
constexpr uint64_t kCounterOffset = 256;
constexpr uint64_t kCutOffset = SECURE_INFER_ATTEND_STATE_BYTES;
static_assert(kCounterOffset + 3 * kMaxGrid * sizeof(uint32_t) <= kCutOffset, "counters");
constexpr uint64_t kSlotOffset = kCutOffset + kMaxGrid * sizeof(Cut);

// One row of n <= 32 partial results, by a warp: lane l gets values 4l .. 4l+3
// of the sum, and all lanes the maximum and the sum of weights.  stats(i):
// where piece i keeps the row's maximum, `sums` floats before its sum;
// values(i): its 128 values.
template <class Stats, class Values>
__device__ __forceinline__ void join_row(int n, Stats stats, int sums, Values values, float4& x, float& top, float& sum)
{
    const int lane = threadIdx.x & 31;
    const float m = lane < n ? __ldcg(stats(lane)) : -INFINITY, l = lane < n ? __ldcg(stats(lane) + sums) : 0.0f;
    x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // The first values are on their way while the weights are found.
    constexpr int kBatch = 6;
    float4 y[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
        if (i < n) y[i] = __ldcg(reinterpret_cast<const float4*>(values(i)) + lane);
    top = m;
    for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    const float f = join_weight(m, top);
    sum = lane < n ? f * l : 0.0f;
    for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    for (int i0 = 0; i0 < n; i0 += kBatch) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (i0 + i >= n) break;
            const float w = __shfl_sync(0xffffffffu, f, i0 + i);
            x.x += w * y[i].x;
            x.y += w * y[i].y;
            x.z += w * y[i].z;
            x.w += w * y[i].w;
            if (i0 + kBatch + i < n) y[i] = __ldcg(reinterpret_cast<const float4*>(values(i0 + kBatch + i)) + lane);
        }
    }
}

// ---------------------------------------------------------------- few rows
//
// Single tokens and short drafts: tiles of eight rows of a KV head, bound by
// reading K and V once.  One CTA per SM; a producer warp keeps three pages
// (64 KiB each, K and V) in flight by TMA.  Each of eight warps takes 16 keys of
// each page, with its own running maximum and sum, so no warp waits for another
// inside the loop.  The products are m16n8k16 with the keys (then the values of
// a head) as M and eight rows as N: a group of eight query heads or fewer fills
// one N, where rows as M would pad them to sixteen, and these instructions are
// slow enough here to matter (about 20 clocks of a quarter SM; with the rows as
// M a batch took 76 us that takes 64 now).  The results join in shared memory
// at the tile's end, and a tile cut over several CTAs is joined by the last of
// them to finish, in the order of the cuts, so results do not depend on the
// order of arrival.
//
// Measured: 47 sequences of up to 8192 tokens, 7 query heads on each of 4 KV
// heads, 65 us, 5.5 TB/s; one sequence of 131072 tokens on one KV head 23 us,
// 2.9 TB/s (three levels of latency before the first page, two joins after the
// last); one of 200 tokens on 8 KV heads 6.7 us.
constexpr int kRowsWarps = 8;
constexpr int kRowsThreads = 32 * (kRowsWarps + 1);
constexpr int kRowsStages = 3;
constexpr int kQuarter = 32;                              // tokens of one TMA box
constexpr uint32_t kQuarterBytes = kQuarter * kDim * 2;   // [2 halves][32 tokens][64 values]
constexpr uint32_t kPageTile = 4 * kQuarterBytes;         // K or V of one page and head
constexpr int kRows = 8;
constexpr uint32_t kRowsSmem = 1024 + kRowsStages * 2 * kPageTile + kRows * 256 + 2 * kRowsWarps * kRows * 4;
// Units up to which a tile is not cut where there is little work.  One sequence
// of 200 tokens: 6.7 us in whole tiles, 7.9 cut; of 512: 8.4 and 8.1.
constexpr int kRowsWhole = 4;
constexpr int kRowsCost = 1;   // pages that a tile's end is worth
// Rows of partial results (512 bytes each) that one CTA joins: reading 80 KiB takes it about as long as counting once
// more in a second step.
constexpr int kJoinRows = 160;
// Partial result of a CTA: [rows][128] sums, [rows] maxima, [rows] sums.
constexpr int kRowSlot = kRows * (kDim + 2);

constexpr int kTilesCost = 2;   // pages that a pair of tiles' beginning and end are worth

// An SM takes 1.1 us of a page for few rows where fewer than 120 of 148 SMs read (58 GB/s each; 120 to 130 get nearly
// all that memory gives), and 1.95 us of a page for a pair of tiles.
__device__ __forceinline__ Kind rows_kind() { return {kRows, kRowsCost, kRowsWhole, 4, 14}; }
__device__ __forceinline__ Kind tiles_kind(const AttendParams& p) { return {2 * (128 / p.group * p.group), kTilesCost, 0, 7, 16}; }

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// An 8 x 8 block of pairs of 16-bit values, transposed over the warp.
__device__ __forceinline__ uint32_t transposed(uint32_t x)
{
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// Barrier of the eight computing warps.
__device__ __forceinline__ void rows_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kRowsWarps) : "memory"); }
// And whether any of their threads says so.
__device__ __forceinline__ bool rows_any(bool x)
{
    uint32_t r;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.aligned.pred q, 1, %2, p;\n selp.u32 %0, 1, 0, q;\n}"
                 : "=r"(r)
                 : "r"(static_cast<uint32_t>(x)), "n"(32 * kRowsWarps)
                 : "memory");
    return r != 0;
}

template <typename T>
__global__ void __launch_bounds__(kRowsThreads, 1)
paged_attend_rows_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                         const __grid_constant__ AttendParams p)
{
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[3 * kRowsStages];   // K full, V full, empty
    __shared__ Share share;
    __shared__ int32_t warp_sums[3 * kRowsThreads / 32];
    __shared__ volatile int stop[2];   // a wait ran out, and work that lets waits go on
    __shared__ int irregular, last_piece;

    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t k_smem = smem_addr(base), v_smem = k_smem + kRowsStages * kPageTile;
    const uint32_t q_smem = v_smem + kRowsStages * kPageTile;
    uint8_t* q_bytes = base + 2 * kRowsStages * kPageTile;
    float* join_m = reinterpret_cast<float*>(q_bytes + kRows * 256);
    float* join_l = join_m + kRowsWarps * kRows;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto k_full = [&](int s) { return smem_addr(&bars[s]); };
    auto v_full = [&](int s) { return smem_addr(&bars[kRowsStages + s]); };
    auto empty = [&](int s) { return smem_addr(&bars[2 * kRowsStages + s]); };
    if (tid == 0) {
        for (int s = 0; s < kRowsStages; ++s) {
            barrier_init(k_full(s), 1);
            barrier_init(v_full(s), 1);
            barrier_init(empty(s), kRowsWarps);
        }
        stop[0] = stop[1] = 0;
        irregular = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
    }
    wait_for_earlier_kernels();
    find_share<kRowsThreads>(p, rows_kind(), tiles_kind(p), &share, warp_sums);
    dependents_may_launch();
    Walk w = start_walk(p, kRows, kRowsCost, share);

    if (warp == kRowsWarps) {
        // Producer: the quarters of each page that hold keys any row sees.
        uint32_t unit = 0, issued = 0;   // units passed, and those whose copies were issued
        while (w.left > 0 && !__any_sync(0xffffffffu, stop[0] || share.down)) {
            const int pages = w.take();
            const int32_t* row = p.table + w.s * p.table_stride + w.span.first + w.page;
            for (int i0 = 0; i0 < pages; i0 += 32) {
                const int id = i0 + lane < pages && w.span.hi > 0 ? row[i0 + lane] : -1;
                for (int i = i0; i < min(pages, i0 + 32); ++i, ++unit) {
                    const int page = __shfl_sync(0xffffffffu, id, i - i0);
                    const int stage = unit % kRowsStages;
                    const uint32_t turn = unit / kRowsStages;
                    if (lane != 0 || stop[0] || (turn > 0 && !barrier_wait(empty(stage), (turn - 1) & 1, stop))) continue;
                    issued = unit + 1;
                    const int first = (w.span.first + w.page + i) * kPage;
                    const int qa = max(0, w.span.lo - first) / kQuarter;
                    const int qb = (min(kPage, w.span.hi - first) + kQuarter - 1) / kQuarter;
                    const uint32_t bytes = qb > qa ? (qb - qa) * kQuarterBytes : 0;
                    barrier_expect(k_full(stage), bytes);
                    for (int t = qa; t < qb; ++t)
                        tma_load_page(k_smem + stage * kPageTile + t * kQuarterBytes, &k_map, k_full(stage),
                                      t * kQuarter, 0, w.head, page);
                    barrier_expect(v_full(stage), bytes);
                    for (int t = qa; t < qb; ++t)
                        tma_load_page(v_smem + stage * kPageTile + t * kQuarterBytes, &v_map, v_full(stage),
                                      t * kQuarter, 0, w.head, page);
                }
                __syncwarp();
            }
            w.advance(p, pages);
        }
        // Copies still in flight land before the CTA's shared memory goes away.
        if (lane == 0) {
            for (uint32_t u = issued > kRowsStages ? issued - kRowsStages : 0; u < issued; ++u) {
                barrier_drain(k_full(u % kRowsStages), (u / kRowsStages) & 1);
                barrier_drain(v_full(u % kRowsStages), (u / kRowsStages) & 1);
            }
        }
        return;
    }

    uint32_t unit = 0;
    // A wait ran out: the rows that are left become NaN, and so do the pieces of cut tiles, which go on being counted.
    // If it was in an earlier call, counts mean nothing and the rows of every piece are written.
    bool failed = share.down != 0;
    while (w.left > 0) {
        const int pages = w.take();
        // The tile's rows, 256 bytes each, in 16-byte pieces swizzled against bank conflicts.
        const int r0 = w.tile * kRows;
        for (int c = tid; c < kRows * 16; c += 32 * kRowsWarps) {
            const int r = c >> 4, piece = c & 15;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (r < w.rows) {
                const int token = (r0 + r) / p.group, g = (r0 + r) % p.group;
                x = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + (w.q.q0 + token) * p.q_token +
                                                    (w.head * p.group + g) * p.q_head + piece * 8);
            }
            *reinterpret_cast<uint4*>(q_bytes + r * 256 + ((piece ^ (r & 7)) << 4)) = x;
        }
        const int cta0 = share.owner(w.tile_unit), cta1 = share.owner(w.tile_unit + w.span.pages - 1);
        const bool split = cta1 > cta0 && !share.down;
        float* slot = p.row_slots + static_cast<int64_t>(2 * blockIdx.x + (static_cast<int>(blockIdx.x) == cta0)) * kRowSlot;
        int lo[2], hi[2];   // keys that this thread's rows see
        int all_lo, all_hi; // keys that every row of the tile sees
        {
            int unused;
            row_keys(p, w.q, w.last_token, all_lo, unused);
            row_keys(p, w.q, w.first_token, unused, all_hi);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = (lane & 3) * 2 + e;
            row_keys(p, w.q, min(w.last_token, (r0 + r) / p.group), lo[e], hi[e]);
        }
        // Sums of values: o[j] holds values 16 j + lane / 4 (+ 8) of rows 2 (lane % 4) (+ 1).
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[j][c] = 0.0f;
        rows_sync();
        uint32_t q[4][4];   // 32 values of the rows each
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const int r = lane & 7, piece = d * 4 + (lane >> 3);
            ldmatrix4(q[d], q_smem + r * 256 + ((piece ^ r) << 4));
        }

        for (int i = 0; i < pages && !failed; ++i, ++unit) {
            const int stage = unit % kRowsStages;
            const uint32_t parity = unit / kRowsStages & 1;
            const int key0 = (w.span.first + w.page + i) * kPage + warp * 16;   // of this warp's keys
            failed = !barrier_wait(k_full(stage), parity, stop) || !barrier_wait(v_full(stage), parity, stop);
            if (failed) break;
            if (key0 < w.span.hi && key0 + 16 > w.span.lo) {
                const uint32_t slice = stage * kPageTile + (warp >> 1) * kQuarterBytes + (warp & 1) * 16 * 128;
                const bool whole = key0 >= all_lo && key0 + 15 <= all_hi;
                float s[2][4] = {};   // two chains of products
#pragma unroll
                for (int d = 0; d < 8; ++d) {   // 16 values of the head at a time
                    uint32_t a[4];
                    const int key = lane & 15, chunk = (d & 3) * 2 + (lane >> 4);
                    ldmatrix4(a, k_smem + slice + (d >> 2) * (kQuarterBytes / 2) + key * 128 + ((chunk ^ (key & 7)) << 4));
                    mma16816<T>(s[d & 1], a, q[d >> 1][(d & 1) * 2], q[d >> 1][(d & 1) * 2 + 1]);
                }
                float x[4], top[2] = {m[0], m[1]};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    x[c] = (s[0][c] + s[1][c]) * p.scale_log2;
                    if (!whole) {
                        const int key = key0 + (lane >> 2) + (c >> 1) * 8;
                        if (key < lo[c & 1] || key > hi[c & 1]) x[c] = -INFINITY;
                    }
                    top[c & 1] = fmaxf(top[c & 1], x[c]);
                }
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], d));
                    top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], d));
                }
                if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float f = m[e] == top[e] ? 1.0f : exp2_approx(m[e] - top[e]);
                        m[e] = top[e];
                        l[e] *= f;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            o[j][e] *= f;
                            o[j][e + 2] *= f;
                        }
                    }
                }
                const float base0 = top[0] == -INFINITY ? 0.0f : top[0], base1 = top[1] == -INFINITY ? 0.0f : top[1];
                const float e0 = exp2_approx(x[0] - base0), e1 = exp2_approx(x[1] - base1);
                const float e2 = exp2_approx(x[2] - base0), e3 = exp2_approx(x[3] - base1);
                l[0] += e0 + e2;
                l[1] += e1 + e3;
                // Weights are rounded to the cache's type for the product; their sum is not.  Keys by rows become rows
                // by keys.
                const uint32_t weight0 = transposed(pack2<T>(e0, e1)), weight1 = transposed(pack2<T>(e2, e3));
                uint32_t keep[2] = {0, 0};   // values of keys that some row sees: this lane's keys 2t, 2t + 1, and 8 more
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = key0 + (j >> 1) * 8 + (lane & 3) * 2 + (j & 1);
                    if (key >= w.span.lo && key < w.span.hi) keep[j >> 1] |= (j & 1) ? 0xffff0000u : 0x0000ffffu;
                }
                uint32_t odd = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint32_t a[4];
                    const int key = (lane & 7) + ((lane >> 4) << 3), chunk = (j & 3) * 2 + ((lane >> 3) & 1);
                    ldmatrix4_trans(a, v_smem + slice + (j >> 2) * (kQuarterBytes / 2) + key * 128 + ((chunk ^ (key & 7)) << 4));
                    if (!whole) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            a[c] &= keep[c >> 1];
                            odd = zero_sum<T>(odd, a[c]);
                        }
                    }
                    mma16816<T>(o[j], a, weight0, weight1);
                }
                if (!whole && w.first_token != w.last_token && zero_sum_odd<T>(odd)) irregular = 1;
            }
            __syncwarp();
            if (lane == 0 && i + 1 < pages) barrier_arrive(empty(stage));
        }

        // Join the warps' results where the last page lay: its buffers are given back afterwards.
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
            if (lane < 4) {
                join_m[warp * kRows + lane * 2 + e] = m[e];
                join_l[warp * kRows + lane * 2 + e] = l[e];
            }
        }
        failed = rows_any(failed);
        const int last_stage = (unit - 1) % kRowsStages;
        const bool by_definition = irregular != 0;
        // Warp i's [8 rows][128] floats, columns swizzled by the row against bank conflicts.
        auto joined = [&](int i) { return base + last_stage * kPageTile + i * 4096; };
        if (!failed) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int r = (lane & 3) * 2 + (c & 1), d = j * 16 + (lane >> 2) + (c >> 1) * 8;
                    *reinterpret_cast<float*>(joined(warp) + r * 512 + (d ^ ((lane & 3) << 3)) * 4) = o[j][c];
                }
        }
        rows_sync();
        // A warp per row.
        if (const int r = warp; r < w.rows) {
            const int token = (r0 + r) / p.group, g = (r0 + r) - token * p.group;
            int a, b;
            row_keys(p, w.q, token, a, b);
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float top, sum;
            if (failed) {
                top = 0.0f;
                sum = NAN;
                x = make_float4(NAN, NAN, NAN, NAN);
            } else if (by_definition) {
                const int ka = (w.span.first + w.page) * kPage;
                row_by_definition<T>(p, static_cast<const T*>(p.q) + (w.q.q0 + token) * p.q_token +
                                            (w.head * p.group + g) * p.q_head,
                                     p.table + w.s * p.table_stride, w.head, max(a, ka), min(b + 1, ka + pages * kPage), top,
                                     sum, x, stop + 1);
            } else {
                const int stat = (lane & (kRowsWarps - 1)) * kRows + r;
                const float mi = join_m[stat];
                top = mi;
#pragma unroll
                for (int d = 1; d < kRowsWarps; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float f = join_weight(mi, top);
                sum = f * join_l[stat];
#pragma unroll
                for (int d = 1; d < kRowsWarps; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
#pragma unroll
                for (int i = 0; i < kRowsWarps; ++i) {
                    const float wi = __shfl_sync(0xffffffffu, f, i);
                    const float4 y = *reinterpret_cast<const float4*>(joined(i) + r * 512 + ((lane * 4) ^ ((r >> 1 & 3) << 3)) * 4);
                    x.x += wi * y.x;
                    x.y += wi * y.y;
                    x.z += wi * y.z;
                    x.w += wi * y.w;
                }
            }
            if (split) {
                *reinterpret_cast<float4*>(slot + r * kDim + lane * 4) = x;
                if (lane == 0) {
                    slot[kRows * kDim + r] = top;
                    slot[kRows * kDim + kRows + r] = sum;
                }
            } else {
                const float inv = 1.0f / sum;
                const int64_t at = static_cast<int64_t>(w.q.q0 + token) * p.heads * p.group + w.head * p.group + g;
                uint2 packed = make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
                if (b < a) packed = make_uint2(0, 0);
                *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at * kDim + lane * 4) = packed;
                if (p.lse != nullptr && lane == 0)
                    p.lse[at] = b >= a ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
            }
        }
        // Reads and writes of this page's buffers come before the next copy into them.
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0 && !failed) barrier_arrive(empty(last_stage));

        if (split) {
            // Piece i of the tile is CTA cta0 + i's.  The last CTA to finish joins them; where that is much to read for
            // one CTA, in two steps: the last of each group of neighbours joins these into its first, the last group
            // those.  Either way in the order of the pieces.
            const int pieces = cta1 - cta0 + 1, mine = static_cast<int>(blockIdx.x) - cta0;
            auto slot_of = [&](int i) { return p.row_slots + static_cast<int64_t>(2 * (cta0 + i) + (i == 0)) * kRowSlot; };
            int group = pieces;
            if (pieces * w.rows > kJoinRows || pieces > 32) {
                group = 2;
                while (group * group < pieces) ++group;
            }
            int first = mine / group * group, n = min(group, pieces - first), step = 1;
            uint32_t* counter = &p.counters[2 * (cta0 + first) + (first == 0)];
            for (;;) {
                __threadfence();
                rows_sync();
                if (tid == 0) last_piece = atomicInc(counter, n - 1) == static_cast<uint32_t>(n - 1);
                rows_sync();
                if (!last_piece) break;
                __threadfence();
                const bool final = step > 1 || n == pieces;
                if (const int r = warp; r < w.rows) {
                    float4 x;
                    float top, sum;
                    join_row(
                        n, [&](int i) { return slot_of(first + i * step) + kRows * kDim + r; }, kRows,
                        [&](int i) { return slot_of(first + i * step) + r * kDim; }, x, top, sum);
                    if (!final) {
                        float* to = slot_of(first);
                        *reinterpret_cast<float4*>(to + r * kDim + lane * 4) = x;
                        if (lane == 0) {
                            to[kRows * kDim + r] = top;
                            to[kRows * kDim + kRows + r] = sum;
                        }
                    } else {
                        const int token = (r0 + r) / p.group, g = (r0 + r) % p.group;
                        int a, b;
                        row_keys(p, w.q, token, a, b);
                        const float inv = 1.0f / sum;
                        const int64_t at = static_cast<int64_t>(w.q.q0 + token) * p.heads * p.group + w.head * p.group + g;
                        uint2 packed = make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
                        if (b < a) packed = make_uint2(0, 0);
                        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at * kDim + lane * 4) = packed;
                        if (p.lse != nullptr && lane == 0)
                            p.lse[at] = b >= a ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
                    }
                }
                if (final) break;
                first = 0;
                step = group;
                n = (pieces + group - 1) / group;
                counter = &p.counters[2 * kMaxGrid + cta0];
            }
        }
        if (by_definition) {
            rows_sync();
            if (tid == 0) irregular = 0;
        }
        rows_sync();
        w.advance(p, pages);
    }
    if (failed && tid == 0) atomicOr(p.status, 1u);
}

// --------------------------------------------------------------- many rows
//
// Chunks: both products on the tcgen05 tensor cores.  One CTA per SM takes two
// tiles of up to 128 rows (whole tokens) that share every page.  A warp loads
// pages by TMA through a ring of four 32 KiB buffers, a warp per tile issues its
// products, and sixteen warps do both tiles' softmax in turn: scores from tensor
// memory, maximum, weights back over the scores in the cache's type, from where
// the second product reads them.  While one tile's softmax runs the other's
// products do.  The accumulated values are only rescaled when a row's maximum
// grew by more than 2^8 since the last time; weights up to 2^8 are as exact as
// weights up to 1, and the sums are 32-bit.  Tensor memory: scores (and weights)
// of the tiles at columns 0 and 128, values at 256 and 384.
//
// For a page and both tiles the tensor cores need 2048 clocks and the special
// function units as many, a quarter fewer as exponentials go to the multiply-add
// units.  Measured 3380: the softmax takes 1690 a tile, of which 900 are the
// exponentials and the rest what the warps of a quarter SM do together (loading
// scores, agreeing on the maximum, handing weights over).  A piece takes 5 us to
// its first scores and 2.5 to leave.  A chunk of 512 tokens after 6144, 32 query
// heads on 8 KV heads: 63 us with the pages in L2 (850 TFLOP/s), 70 without (768);
// 4096 tokens in 20480: 1.13 to 1.22 ms, 1.0 to 1.09 PFLOP/s, which is the
// products' part of the page loop (2048 of 3380 clocks) at the SM clock of 1.4 GHz
// that such a call runs at.
constexpr int kSoftWarps = 16;       // four warpgroups, each with a quarter of a page's keys
constexpr int kTileThreads = 32 * (kSoftWarps + 4);   // and producer, products of two tiles, guard
constexpr int kRing = 4;
constexpr uint32_t kStageBytes = 32 * 32;   // 32 bytes of a softmax warp's rows, on their way to whole sectors
constexpr uint32_t kTileBytes = 128 * kDim * 2;
constexpr int kItems = 8;
constexpr int kTileRows = 256;
// Partial result of a pair of tiles: the values as tensor memory gives them to a warp, [8 warps' rows][32 fours of
// values][32 rows][4], so that a warp's stores cover whole lines, then [rows] maxima and [rows] sums.  (Row by row, by
// way of shared memory, a piece's end took 2 us more for each tile.)
constexpr int kTileSlot = kTileRows * (kDim + 2);
constexpr float kRescale = 8.0f;

template <int kCols>
__device__ __forceinline__ void tmem_load(uint32_t (&r)[kCols], uint32_t addr);
template <>
__device__ __forceinline__ void tmem_load<32>(uint32_t (&r)[32], uint32_t addr)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
template <>
__device__ __forceinline__ void tmem_load<16>(uint32_t (&r)[16], uint32_t addr)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit_to(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// Two 32-bit values in a register pair.
__device__ __forceinline__ uint64_t pair(uint32_t x, uint32_t y)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(x), "r"(y));
    return r;
}
// Shared-memory operands lie in the 128-byte swizzle, groups of eight 128-byte
// rows 1024 bytes apart.  A descriptor's low word holds the address and, for an
// operand whose rows run along the product's sum (V), the bytes between the two
// halves of 64 values; its high word is the same for all.  Advancing along the
// sum adds to the low word.
constexpr uint32_t kOperandHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t operand(uint32_t addr, uint32_t half) { return (addr >> 4 & 0x3fff) | (half >> 4) << 16; }
__device__ __forceinline__ uint64_t operand_at(uint32_t low, uint32_t bytes) { return pair(low + (bytes >> 4), kOperandHigh); }

template <bool kAdd>
__device__ __forceinline__ void product_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t desc)
{
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
                 "l"(a), "l"(b), "r"(desc), "n"(kAdd)
                 : "memory");
}
__device__ __forceinline__ void product_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, uint32_t accumulate)
{
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
                 "r"(a), "l"(b), "r"(desc), "r"(accumulate)
                 : "memory");
}
// One lane of a converged warp, the same one at every call.
__device__ __forceinline__ bool elected()
{
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
    return r != 0;
}

__device__ __forceinline__ void tma_load_rows(uint32_t dst, const CUtensorMap* map, uint32_t bar, int head, int token, int half)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(0), "r"(head), "r"(token), "r"(half)
        : "memory");
}

__device__ __forceinline__ uint64_t pair(float x, float y) { return pair(__float_as_uint(x), __float_as_uint(y)); }
__device__ __forceinline__ float2 unpair(uint64_t v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 2^x of a pair on the multiply-add units, for x <= 126: x = n + f with n the
// nearest integer, 2^f by the polynomial of degree 4 with the least largest
// relative error on [-1/2, 1/2] (2.7e-6, by Remez's exchange), n added to the
// exponent.  Below -126 it stays at 2^-126, which beside a largest weight of 2^-8
// or more is nothing.  NaN does not survive.
__device__ __forceinline__ float2 exp2_poly(uint64_t x2)
{
    constexpr float kRound = 12582912.0f;   // 1.5 2^23: the sum's last bits are n
    float2 x = unpair(x2);
    x2 = pair(fmaxf(x.x, -126.0f), fmaxf(x.y, -126.0f));
    const uint64_t t = add2(x2, pair(kRound, kRound));
    const uint64_t n = add2(t, pair(-kRound, -kRound));
    const uint64_t f = fma2(n, pair(-1.0f, -1.0f), x2);
    uint64_t y = fma2(pair(0.009570102f, 0.009570102f), f, pair(0.05591786f, 0.05591786f));
    y = fma2(y, f, pair(0.24024744f, 0.24024744f));
    y = fma2(y, f, pair(0.6931218f, 0.6931218f));
    y = fma2(y, f, pair(0.9999993f, 0.9999993f));
    const float2 r = unpair(y), e = unpair(t);
    return make_float2(__uint_as_float(__float_as_uint(r.x) + (__float_as_uint(e.x) << 23)),
                       __uint_as_float(__float_as_uint(r.y) + (__float_as_uint(e.y) << 23)));
}

// A CTA's piece of a tile, from the producer for the other warps.  The producer
// is less than kItems pieces ahead of the last of them: it needs the first
// product of the piece before, and buffers that the guard gives back, who
// waits for every softmax warp.
struct Item {
    Span span;
    int s, head, pages, rows;
    int first_key;               // of the piece
    int pos, last_pos, last_key; // of the tile's first and last token, and of the sequence
    int lo_all, hi_all;          // keys that every row sees
    int q0;                      // the tile's first token among all
    int slot;                    // where a part of a cut tile goes, -1: the tile is whole
    int more;                    // another piece follows

    // Keys that the row at position p sees: [lo, hi].
    __device__ __forceinline__ void keys(const AttendParams& a, int p, int& lo, int& hi) const
    {
        hi = a.causal ? min(last_key, p) : last_key;
        lo = a.window ? max(0, p - a.window + 1) : 0;
    }
};

struct TilesControl {
    uint64_t kv_full[kRing], kv_empty[kRing], q_full, q_empty;
    uint64_t s_full[2], p_ready[2], o_full[2], drained[2];
    uint64_t checked, taken, item_full[kItems];
    Item items[kItems];
    float exchange[2][4][128];           // between a row's four threads
    int32_t warp_sums[3 * kTileThreads / 32];
    Share share;
    uint32_t tmem;
    int irregular;                       // what the guard found in the piece
    int stop[2];                         // a wait ran out, and work that lets waits go on
};
constexpr uint32_t kControlBytes = 8192 - 1024;   // operands follow at the next whole KiB, which the swizzle needs
static_assert(sizeof(TilesControl) <= kControlBytes, "control block");
constexpr uint32_t kTilesSmem = kControlBytes + 1024 + (2 + kRing) * kTileBytes + kSoftWarps * kStageBytes;

// After a wait that ran out, by the softmax warps: the rows of this CTA's share
// become NaN, and so do its pieces of cut tiles.
template <typename T>
__device__ __noinline__ void fail_tiles(const AttendParams& p, const Share& share)
{
    const int tid = threadIdx.x, cta = blockIdx.x;
    if (tid == 0) atomicOr(p.status, 1u);
    Walk w = start_walk(p, 2 * (128 / p.group * p.group), kTilesCost, share);
    for (bool first = true; w.left > 0; first = false) {
        const int pages = w.take();
        const int cta0 = share.owner(w.tile_unit), cta1 = share.owner(w.tile_unit + w.span.pages - 1);
        if (first && tid == 0)
            p.cuts[cta] = cta0 < cta ? Cut{cta1, cta0, w.rows, w.first_token, w.head, w.q.n, w.q.kv, w.q.q0} : Cut{};
        if (cta1 > cta0) {
            float* slot = p.slots + static_cast<int64_t>(2 * cta + (cta0 == cta)) * kTileSlot;
            for (int i = tid; i < kTileSlot; i += 32 * kSoftWarps) slot[i] = NAN;
        } else {
            for (int i = tid; i < w.rows * 32; i += 32 * kSoftWarps) {
                const int r = i >> 5, token = w.first_token + r / p.group;
                const int64_t at = (static_cast<int64_t>(w.q.q0 + token) * p.heads + w.head) * p.group + r % p.group;
                const uint32_t x = pack2<T>(NAN, NAN);
                reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at * kDim)[i & 31] = make_uint2(x, x);
                if (p.lse != nullptr && (i & 31) == 0) p.lse[at] = NAN;
            }
        }
        w.advance(p, pages);
    }
}

template <typename T>
__global__ void __launch_bounds__(kTileThreads, 1)
paged_attend_tiles_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                          const __grid_constant__ CUtensorMap v_map, const __grid_constant__ AttendParams p)
{
    extern __shared__ __align__(16) uint8_t smem_raw[];
    TilesControl& c = *reinterpret_cast<TilesControl*>(smem_raw);
    volatile int* const stop = c.stop;
    const uint32_t q_smem = (smem_addr(smem_raw) + kControlBytes + 1023) & ~1023u, ring = q_smem + 2 * kTileBytes;
    auto kv_full = [&](int i) { return smem_addr(&c.kv_full[i]); };
    auto kv_empty = [&](int i) { return smem_addr(&c.kv_empty[i]); };
    const uint32_t q_full = smem_addr(&c.q_full), q_empty = smem_addr(&c.q_empty);
    auto s_full = [&](int w) { return smem_addr(&c.s_full[w]); };
    auto p_ready = [&](int w) { return smem_addr(&c.p_ready[w]); };
    auto o_full = [&](int w) { return smem_addr(&c.o_full[w]); };
    auto drained = [&](int w) { return smem_addr(&c.drained[w]); };
    auto item_full = [&](uint32_t i) { return smem_addr(&c.item_full[i % kItems]); };
    const uint32_t checked = smem_addr(&c.checked), taken = smem_addr(&c.taken);

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < kRing; ++i) {
            barrier_init(kv_full(i), 1);
            barrier_init(kv_empty(i), 3);    // each tile's products and the guard
        }
        barrier_init(q_full, 1);
        barrier_init(q_empty, 2);
        for (int w = 0; w < 2; ++w) {
            barrier_init(s_full(w), 1);
            barrier_init(p_ready(w), kSoftWarps);
            barrier_init(o_full(w), 1);
            barrier_init(drained(w), 1);
        }
        barrier_init(checked, 1);
        barrier_init(taken, kSoftWarps);
        for (int i = 0; i < kItems; ++i) barrier_init(item_full(i), 1);
        c.stop[0] = c.stop[1] = 0;
        c.irregular = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&q_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
    }
    if (warp == kSoftWarps + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&c.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tmem_fence_before();
    }
    // Beside the kernel for few rows this one starts as that one's CTAs leave: its inputs were complete before that one
    // read them, the two share no memory that either writes, and it waits for that one at its end instead.
    if (!p.both) wait_for_earlier_kernels();
    const int tokens = 128 / p.group, rows_per_tile = tokens * p.group;   // of one of the two tiles
    find_share<kTileThreads>(p, tiles_kind(p), rows_kind(), &c.share, c.warp_sums);
    dependents_may_launch();
    tmem_fence_after();
    const uint32_t tmem = c.tmem;
    Walk w = start_walk(p, 2 * rows_per_tile, kTilesCost, c.share);
    const bool any = w.left > 0 && c.share.down == 0;

    // 640 threads at 96 registers: 104 for the four softmax warpgroups and 64 for the fifth make the same sum.
    if (warp >= kSoftWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == kSoftWarps) {
            // Producer.
            uint32_t n = 0, item = 0, issued = 0, q_issued = 0;   // buffers and pieces passed, and those whose copies were issued
            while (any && w.left > 0 && !__any_sync(0xffffffffu, *stop)) {
                const int pages = w.take();
                const int32_t* row = p.table + w.s * p.table_stride + w.span.first + w.page;
                int id = lane < pages && w.span.hi > 0 ? __ldcg(row + lane) : -1;
                if (lane == 0) {
                    if (item > 0) barrier_wait(q_empty, (item - 1) & 1, stop);
                    if (!*stop) {
                        const int tiles = w.rows > rows_per_tile ? 2 : 1;
                        barrier_expect(q_full, tiles * 2 * rows_per_tile * 128);
                        q_issued = item + 1;
                        for (int t = 0; t < tiles; ++t)
                            for (int h = 0; h < 2; ++h)
                                tma_load_rows(q_smem + t * kTileBytes + h * (kTileBytes / 2), &q_map, q_full,
                                              w.head * p.group, w.q.q0 + w.first_token + t * tokens, h);
                    }
                }
                __syncwarp();
                auto publish = [&] {
                    Item& it = c.items[item % kItems];
                    it.span = w.span;
                    it.s = w.s;
                    it.head = w.head;
                    it.pages = pages;
                    it.rows = w.rows;
                    it.first_key = (w.span.first + w.page) * kPage;
                    it.pos = w.q.kv - w.q.n + w.first_token;
                    it.last_pos = it.pos + w.last_token - w.first_token;
                    it.last_key = w.q.kv - 1;
                    int unused;
                    it.keys(p, it.last_pos, it.lo_all, unused);
                    it.keys(p, it.pos, unused, it.hi_all);
                    it.q0 = w.q.q0 + w.first_token;
                    const int cta0 = c.share.owner(w.tile_unit), cta1 = c.share.owner(w.tile_unit + w.span.pages - 1);
                    it.slot = cta1 > cta0 ? 2 * static_cast<int>(blockIdx.x) + (cta0 == static_cast<int>(blockIdx.x)) : -1;
                    it.more = w.left > pages + w.cost;
                    barrier_arrive(item_full(item));
                    // Only the first tile of a CTA can have begun in an earlier one.
                    if (item == 0) {
                        Cut cut{};
                        if (cta0 < static_cast<int>(blockIdx.x))
                            cut = Cut{cta1, cta0, w.rows, w.first_token, w.head, w.q.n, w.q.kv, w.q.q0};
                        p.cuts[blockIdx.x] = cut;
                    }
                };
                for (int i0 = 0; i0 < pages; i0 += 32) {
                    if (i0 > 0) id = i0 + lane < pages && w.span.hi > 0 ? __ldcg(row + i0 + lane) : -1;
                    for (int i = i0; i < min(pages, i0 + 32); ++i) {
                        const int page = __shfl_sync(0xffffffffu, id, i - i0);
                        for (int kv = 0; kv < 2; ++kv, ++n) {
                            const uint32_t slot = n % kRing, turns = n / kRing;
                            if (lane == 0 && !*stop && (turns == 0 || barrier_wait(kv_empty(slot), (turns - 1) & 1, stop))) {
                                barrier_expect(kv_full(slot), kTileBytes);
                                issued = n + 1;
                                tma_load_page(ring + slot * kTileBytes, kv ? &v_map : &k_map, kv_full(slot), 0, 0, w.head, page);
                            }
                            // The others hear of the piece once its first loads are on their way.
                            if (lane == 0 && i == 0 && kv == 0) publish();
                        }
                    }
                    __syncwarp();
                }
                ++item;
                w.advance(p, pages);
            }
            if (lane == 0) {
                for (uint32_t u = issued > kRing ? issued - kRing : 0; u < issued; ++u) barrier_drain(kv_full(u % kRing), (u / kRing) & 1);
                if (q_issued > 0) barrier_drain(q_full, (q_issued - 1) & 1);
            }
            __syncwarp();
        } else if (warp < kSoftWarps + 3) {
            // Products, a warp per tile.  The softmax warps take the tiles in turn, and so do these.
            const int t = warp - kSoftWarps - 1;
            constexpr uint32_t type = std::is_same<T, __half>::value ? 0u : 1u;
            constexpr uint32_t desc = 1u << 4 | type << 7 | type << 10 | (128u >> 3) << 17 | (128u >> 4) << 24;
            constexpr uint32_t desc_v = desc | 1u << 16;   // V's rows run along the sum
            const uint32_t q = operand(q_smem + t * kTileBytes, 0), s_at = tmem + t * 128, o_at = tmem + 256 + t * 128;
            uint32_t n = 0, item = 0, ready = 0;   // buffers and pieces taken, softmax tiles
            auto scores = [&](uint32_t slot) {
                const uint32_t k = operand(ring + slot * kTileBytes, 0);
                product_smem<false>(s_at, operand_at(q, 0), operand_at(k, 0), desc);
#pragma unroll
                for (int i = 1; i < 8; ++i) {
                    const uint32_t at = (i >> 2) * (kTileBytes / 2) + (i & 3) * 32;
                    product_smem<true>(s_at, operand_at(q, at), operand_at(k, at), desc);
                }
                commit_to(s_full(t));
                commit_to(kv_empty(slot));
            };
            bool ok = true;
            while (ok && any) {
                ok = barrier_wait(item_full(item), (item / kItems) & 1, stop) && barrier_wait(q_full, item & 1, stop);
                if (!ok) break;
                const Item& w = c.items[item % kItems];
                const int pages = w.pages;
                const bool last = !w.more;
                if (t == 1 && w.rows <= rows_per_tile) {
                    // No second tile: its share of the buffers is given back as they fill.
                    for (int i = 0; ok && i < 2 * pages; ++i, ++n) {
                        ok = barrier_wait(kv_full(n % kRing), (n / kRing) & 1, stop);
                        if (ok && lane == 0) barrier_arrive(kv_empty(n % kRing));
                    }
                    if (lane == 0) barrier_arrive(q_empty);
                } else {
                    // Unused rows beside used ones become zero: 32 rows are rescaled together, and the roundings of the
                    // used ones would follow others' queries, or what shared memory held.
                    if (const int used = min(rows_per_tile, w.rows - t * rows_per_tile); used & 31) {
                        const uint32_t end = q_smem + t * kTileBytes + (lane & 8 ? kTileBytes / 2 : 0) + ((used | 31) + 1) * 128;
#pragma unroll 4
                        for (uint32_t at = end - ((used | 31) + 1 - used - (lane >> 4)) * 128 + (lane & 7) * 16; at < end; at += 256)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                    }
                    ok = ok && barrier_wait(kv_full(n % kRing), (n / kRing) & 1, stop);
                    if (!ok) break;
                    tmem_fence_after();
                    if (elected()) {
                        scores(n % kRing);
                        if (pages == 1) commit_to(q_empty);
                    }
                    __syncwarp();
                    ++n;
                    for (int i = 0; i < pages; ++i) {
                        const uint32_t v_slot = n % kRing, k_slot = (n + 1) % kRing;
                        const bool more = i + 1 < pages;
                        ok = barrier_wait(kv_full(v_slot), (n / kRing) & 1, stop);
                        // Values of keys that no row sees were never written or belong to others: weights of zero do
                        // not silence a NaN there, so within the 16-key steps that are multiplied they become zero.
                        const int key0 = w.first_key + i * kPage;
                        const int lo = max(0, min(kPage, w.span.lo - key0)), hi = max(0, min(kPage, w.span.hi - key0));
                        const int step0 = lo >> 4, step1 = hi > lo ? (hi + 15) >> 4 : step0;
                        if (lo & 15 || hi & 15) {
                            for (int side = 0; side < 2; ++side) {
                                const int a = side ? hi : step0 * 16, b = side ? min(kPage, step1 * 16) : lo;
                                for (int x = lane; x < (b - a) * 16; x += 32) {
                                    const uint32_t at = ring + v_slot * kTileBytes + (x & 8 ? kTileBytes / 2 : 0) +
                                                        (a + (x >> 4)) * 128 + (x & 7) * 16;
                                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
                                }
                            }
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                            __syncwarp();
                        }
                        if (ok && more) ok = barrier_wait(kv_full(k_slot), ((n + 1) / kRing) & 1, stop);
                        ok = ok && barrier_wait(p_ready(t), ready & 1, stop);
                        if (!ok) break;
                        ++ready;
                        tmem_fence_after();
                        if (elected()) {
                            const uint32_t v = operand(ring + v_slot * kTileBytes, kTileBytes / 2);
                            if (step0 == 0 && step1 == 8) {
                                product_tmem(o_at, s_at, operand_at(v, 0), desc_v, i > 0);
#pragma unroll
                                for (int k = 1; k < 8; ++k) product_tmem(o_at, s_at + k * 8, operand_at(v, k * 2048), desc_v, 1);
                            } else {
                                // A page that no row sees still sets the values to zero where it is the first.
                                const int s0 = step1 > step0 ? step0 : 0, s1 = step1 > step0 ? step1 : (i == 0 ? 1 : 0);
                                for (int k = s0; k < s1; ++k)
                                    product_tmem(o_at, s_at + k * 8, operand_at(v, k * 2048), desc_v, i > 0 || k > s0);
                            }
                            if (more) scores(k_slot);
                            else commit_to(o_full(t));
                            commit_to(kv_empty(v_slot));
                            if (i + 2 == pages) commit_to(q_empty);
                        }
                        __syncwarp();
                        n += more ? 2 : 1;
                    }
                }
                ++item;
                if (last) break;
            }
            // Nothing of this warp is in flight when tensor memory is given back.
            if (elected()) commit_to(drained(t));
            __syncwarp();
            barrier_drain(drained(t), 0);
        } else {
            // Guard: an infinity or NaN among values that some rows see and others do not, where weights of zero
            // would carry it over.
            uint32_t n = 0, item = 0;
            while (any) {
                if (!barrier_wait(item_full(item), (item / kItems) & 1, stop)) break;
                const Item w = c.items[item % kItems];
                const int pages = w.pages, lo_all = w.lo_all, hi_all = w.hi_all;
                uint32_t odd = 0;
                for (int i = 0; i < pages; ++i) {
                    const int key0 = w.first_key + i * kPage;
                    for (int kv = 0; kv < 2; ++kv, ++n) {
                        const uint32_t slot = n % kRing;
                        if (!barrier_wait(kv_full(slot), (n / kRing) & 1, stop)) break;
                        if (kv == 1 && w.pos != w.last_pos && (key0 < lo_all || key0 + kPage - 1 > hi_all)) {
                            // Two keys at a time: left of what all rows see, then right of it.
                            const int a = max(0, w.span.lo - key0), b = min(kPage, w.span.hi - key0);
                            for (int side = 0; side < 2; ++side) {
                                const int k0 = side ? max(a, hi_all + 1 - key0) : a, k1 = side ? b : min(b, lo_all - key0);
                                const uint32_t at = ring + slot * kTileBytes + (lane & 8 ? kTileBytes / 2 : 0) + (lane & 7) * 16;
#pragma unroll 8
                                for (int key = k0 + (lane >> 4); key < k1; key += 2) {
                                    uint4 x;
                                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                                                 : "r"(at + key * 128));
                                    odd = zero_sum<T>(zero_sum<T>(zero_sum<T>(zero_sum<T>(odd, x.x), x.y), x.z), x.w);
                                }
                            }
                        }
                        __syncwarp();
                        if (lane == 0) barrier_arrive(kv_empty(slot));
                    }
                }
                // The flag is the previous item's until the softmax has read it.
                if (item > 0) barrier_wait(taken, (item - 1) & 1, stop);
                const bool found = __any_sync(0xffffffffu, zero_sum_odd<T>(odd));
                if (lane == 0) c.irregular = found;
                __syncwarp();
                if (lane == 0) barrier_arrive(checked);
                ++item;
                if (!w.more) break;
            }
        }
    } else {
        // Softmax: a row by four threads, each with a quarter of a page's keys, the tiles in turn: while one tile's
        // products run all warps are at the other.  After a wait that ran out the loops run on without waiting to the
        // piece's end, so the four keep meeting, and leave it together.
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        const int quarter = warp >> 2, rows0 = (warp & 3) * 32, row = rows0 + lane;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);
        const float scale = fabsf(p.scale_log2);
        const bool flip = p.scale_log2 < 0.0f;
        // The four warps that hold the same 32 rows: whether any of their threads says so.
        auto meet_or = [&](bool x) {
            uint32_t r;
            asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n barrier.cta.red.or.aligned.pred q, %1, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
                         : "=r"(r)
                         : "r"(1 + (warp & 3)), "r"(static_cast<uint32_t>(x))
                         : "memory");
            return r != 0;
        };
        const int token = row / p.group, g = row % p.group;   // within the tile
        const int rel = token * p.heads * p.group + g;        // rows of the output from the tile's first
        uint32_t seen[2] = {0, 0}, done[2] = {0, 0}, item = 0;   // completions of s_full and o_full taken
        bool ok = true;
        while (any) {
            ok = ok && barrier_wait(item_full(item), (item / kItems) & 1, stop);
            if (meet_or(!ok)) break;
            const Item& w = c.items[item % kItems];
            const int pages = w.pages, tiles = w.rows > rows_per_tile ? 2 : 1;
            const int lo_all = w.lo_all, hi_all = w.hi_all, page_key = w.first_key;
            float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
            for (int i = 0; i < pages; ++i) {
                // By the whole page and both tiles, so that all threads agree.
                const int page0 = page_key + i * kPage;
                const bool masked = page0 < lo_all || page0 + kPage - 1 > hi_all;
#pragma unroll 1
                for (int t = 0; t < tiles; ++t) {
                    ok = ok && barrier_wait(s_full(t), (t ? seen[1] : seen[0]) & 1, stop);
                    if (t) ++seen[1];
                    else ++seen[0];
                    tmem_fence_after();
                    float m = t ? m1 : m0, l = t ? l1 : l0;
                    const uint32_t s_at = lanes + t * 128 + quarter * 32, w_at = lanes + t * 128 + quarter * 16;
                    bool fresh = i == 0 || masked || flip;
                    if (!fresh) {
                        // The usual page: weights by the maximum so far, while the page's own is found.
                        uint32_t s[32], w2[16];
                        tmem_load<32>(s, s_at);
                        tmem_wait_loads();
                        const float base = m == -INFINITY ? 0.0f : m * scale;
                        const uint64_t scale2 = pair(scale, scale), base2 = pair(-base, -base);
                        uint64_t sum[2] = {};
                        float tops[2] = {m, m};
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const uint64_t x = fma2(pair(s[2 * j], s[2 * j + 1]), scale2, base2);
                            tops[j & 1] = max3_nan(tops[j & 1], __uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1]));
                            float2 e;
                            // A quarter of the exponentials go to the multiply-add units, which levels these with the
                            // special function units.
                            if (j % 4 == 1) {
                                e = exp2_poly(x);
                            } else {
                                const float2 y = unpair(x);
                                e = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                            }
                            sum[j & 1] = add2(sum[j & 1], pair(e.x, e.y));
                            // Weights are rounded to the cache's type for the product; their sum is not.
                            w2[j] = pack2<T>(e.x, e.y);
                        }
                        const float top = max3_nan(tops[0], tops[1], tops[1]);
                        // Weights may cover scores once the row's other threads have read theirs.
                        tmem_fence_before();
                        // (A row that has only met scores of minus infinity is not for the polynomial either.)
                        fresh = meet_or(!((top - m) * scale <= kRescale));
                        tmem_fence_after();
                        if (!fresh) {
                            tmem_store(w_at, w2);
                            const float2 sums = unpair(add2(sum[0], sum[1]));
                            l += sums.x + sums.y;
                        }
                    }
                    if (fresh) {
                        // The first page, one whose mask hides keys, or one that some row's maximum outgrew.
                        uint32_t s[32];
                        tmem_load<32>(s, s_at);
                        tmem_wait_loads();
                        if (flip) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) s[j] ^= 0x80000000u;
                        }
                        if (masked) {
                            // Bits of the keys from lo to hi.
                            int lo, hi;
                            w.keys(p, min(w.pos + t * tokens + token, w.last_pos), lo, hi);
                            const int a = max(0, lo - page0 - quarter * 32), b = min(31, hi - page0 - quarter * 32);
                            const uint32_t keep = b < a ? 0 : (~0u << a) & (~0u >> (31 - b));
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (!(keep >> j & 1)) s[j] = 0xff800000u;
                        }
                        float tops[2] = {m, m};
#pragma unroll
                        for (int j = 0; j < 32; j += 2)
                            tops[(j >> 1) & 1] = max3_nan(tops[(j >> 1) & 1], __uint_as_float(s[j]), __uint_as_float(s[j + 1]));
                        float top = max3_nan(tops[0], tops[1], tops[1]);
                        // And the row's other threads'.
                        c.exchange[t][quarter][row] = top;
                        tmem_fence_before();
                        meet_or(false);
                        tmem_fence_after();
                        const float* others = &c.exchange[t][0][row];
                        top = max3_nan(max3_nan(others[0], others[128], others[256]), others[384], top);
                        if (top == INFINITY) top = NAN;   // a NaN or infinite score makes its row NaN
                        if (i == 0) {
                            m = top;
                        } else if (__any_sync(0xffffffffu, !((top - m) * scale <= kRescale) && top != -INFINITY)) {
                            const float f = m == top ? 1.0f : exp2_approx((m - top) * scale);
                            l *= f;
                            const uint32_t o_at = lanes + 256 + t * 128 + quarter * 32;
#pragma unroll 1
                            for (int d = 0; d < 32; d += 16) {
                                uint32_t o[16];
                                tmem_load<16>(o, o_at + d);
                                tmem_wait_loads();
#pragma unroll
                                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                                tmem_store(o_at + d, o);
                            }
                            m = top;
                        }
                        const float base = m == -INFINITY ? 0.0f : m * scale;
                        float sum[2] = {};
                        uint32_t w2[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float e0 = exp2_approx(fmaf(__uint_as_float(s[2 * j]), scale, -base));
                            const float e1 = exp2_approx(fmaf(__uint_as_float(s[2 * j + 1]), scale, -base));
                            sum[j & 1] += e0 + e1;
                            w2[j] = pack2<T>(e0, e1);
                        }
                        tmem_store(w_at, w2);
                        l += sum[0] + sum[1];
                    }
                    if (t) m1 = m, l1 = l;
                    else m0 = m, l0 = l;
                    tmem_wait_stores();
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0) barrier_arrive(p_ready(t));
                }
            }
            ok = ok && barrier_wait(checked, item & 1, stop);
            ok = !meet_or(!ok);   // the four go the same way
            const bool split = w.slot >= 0, by_definition = ok && *static_cast<volatile int*>(&c.irregular) != 0;
            float* slot = p.slots + static_cast<int64_t>(w.slot) * kTileSlot;
            const uint32_t stage = ring + kRing * kTileBytes + warp * kStageBytes;
#pragma unroll 1
            for (int t = 0; t < tiles; ++t) {
                ok = ok && barrier_wait(o_full(t), (t ? done[1] : done[0]) & 1, stop);
                if (t) ++done[1];
                else ++done[0];
                tmem_fence_after();
                // Output row of the tile's first row, and how many of the warp's rows are used.
                const int64_t out0 = static_cast<int64_t>(w.q0 + t * tokens) * p.heads * p.group + w.head * p.group;
                const int valid = min(rows_per_tile, w.rows - t * rows_per_tile) - rows0;
                if (by_definition) {
                    for (int r = quarter; r < min(32, valid); r += 4) {
                        const int tok = (rows0 + r) / p.group, head = (rows0 + r) % p.group;
                        int a, b;
                        w.keys(p, w.pos + t * tokens + tok, a, b);
                        float mm, ll;
                        float4 x;
                        row_by_definition<T>(p, static_cast<const T*>(p.q) + (w.q0 + t * tokens + tok) * p.q_token +
                                                    (w.head * p.group + head) * p.q_head,
                                             p.table + w.s * p.table_stride, w.head, max(a, page_key),
                                             min(b + 1, page_key + pages * kPage), mm, ll, x, stop + 1);
                        if (split) {
                            reinterpret_cast<float4*>(slot)[((t * 4 + rows0 / 32) * 32 + lane) * 32 + r] = x;
                            if (lane == 0) {
                                slot[kTileRows * kDim + t * 128 + rows0 + r] = mm;
                                slot[kTileRows * kDim + kTileRows + t * 128 + rows0 + r] = ll;
                            }
                        } else {
                            const float inv = 1.0f / ll;
                            const int64_t at = out0 + tok * p.heads * p.group + head;
                            uint2 packed = make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
                            if (b < a) packed = make_uint2(0, 0);
                            *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at * kDim + lane * 4) = packed;
                            if (p.lse != nullptr && lane == 0)
                                p.lse[at] = b >= a ? (mm + log2f(ll)) * 0.6931471805599453f : -INFINITY;
                        }
                    }
                    continue;
                }
                c.exchange[t][quarter][row] = t ? l1 : l0;
                meet_or(false);
                const float* parts = &c.exchange[t][0][row];
                const float l = (parts[0] + parts[128]) + (parts[256] + parts[384]);
                meet_or(false);   // read before the next piece's maxima come
                int lo, hi;
                w.keys(p, min(w.pos + t * tokens + token, w.last_pos), lo, hi);
                const float inv = 1.0f / l;
                // Rows leave through a warp's own piece of shared memory, 32 bytes of each at a time, so that a store
                // covers whole sectors: sixteen rows by two lanes.
                auto put = [&](uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, int j) {
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 32 + ((j ^ (lane >> 2 & 1)) << 4)),
                                 "r"(x0), "r"(x1), "r"(x2), "r"(x3)
                                 : "memory");
                };
                auto get = [&](int r) {
                    uint4 x;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                                 : "r"(stage + r * 32 + (((lane & 1) ^ (r >> 2 & 1)) << 4))
                                 : "memory");
                    return x;
                };
                uint32_t o[32];
                tmem_load<32>(o, lanes + 256 + t * 128 + quarter * 32);
                tmem_wait_loads();
                if (split) {
                    float4* part = reinterpret_cast<float4*>(slot) + ((t * 4 + rows0 / 32) * 32 + quarter * 8) * 32 + lane;
                    if (lane < valid) {
#pragma unroll
                        for (int d = 0; d < 32; d += 4)
                            part[d * 8] = make_float4(__uint_as_float(o[d]), __uint_as_float(o[d + 1]),
                                                      __uint_as_float(o[d + 2]), __uint_as_float(o[d + 3]));
                    }
                } else {
                    T* out = static_cast<T*>(p.out) + out0 * kDim + quarter * 32 + (lane & 1) * 8;
#pragma unroll
                    for (int d = 0; d < 32; d += 16) {
                        uint32_t x[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            x[j] = hi >= lo ? pack2<T>(__uint_as_float(o[d + 2 * j]) * inv, __uint_as_float(o[d + 2 * j + 1]) * inv) : 0u;
                        put(x[0], x[1], x[2], x[3], 0);
                        put(x[4], x[5], x[6], x[7], 1);
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int r = k * 16 + (lane >> 1);
                            const int64_t to = __shfl_sync(0xffffffffu, rel, r);
                            const uint4 y = get(r);
                            if (r < valid) *reinterpret_cast<uint4*>(out + to * kDim + d) = y;
                        }
                        __syncwarp();
                    }
                }
                if (lane < valid && quarter == 0) {
                    const float top = (t ? m1 : m0) * scale;
                    if (split) {
                        slot[kTileRows * kDim + t * 128 + row] = top;
                        slot[kTileRows * kDim + kTileRows + t * 128 + row] = l;
                    } else if (p.lse != nullptr) {
                        p.lse[out0 + rel] = hi >= lo ? (top + log2f(l)) * 0.6931471805599453f : -INFINITY;
                    }
                }
                tmem_fence_before();
            }
            const bool last = !w.more;
            ++item;
            __syncwarp();
            if (lane == 0) barrier_arrive(taken);
            if (last) break;
        }
        if (tid == 0 && !any) p.cuts[blockIdx.x] = Cut{};
    }
    tmem_fence_before();
    __syncthreads();
    if (warp < kSoftWarps && (*stop || c.share.down)) fail_tiles<T>(p, c.share);
    if (p.both) wait_for_earlier_kernels();
    if (warp == kSoftWarps + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// Joins the pieces of tiles that were cut over CTAs, in the order of the pieces.
// A lane takes a row, as the pieces lie, and kFours times four of its values;
// the blocks of the CTAs that went on with a tile share its values, so a tile
// in many pieces has more warps.  Bound by reading the pieces from L2 and by
// latency, so all blocks are there at once: two warps each (eight, with four of
// them on a value's pieces, had to take turns: 10 us more where every CTA ends a
// tile).
constexpr int kJoinThreads = 64;
constexpr int kJoinBlocks = kTileRows / 32 * (kDim / 16) / (kJoinThreads / 32);
template <typename T, int kFours>
__device__ __forceinline__ void join_values(const AttendParams& p, const Cut& cut, int r, int tile_row, int d4)
{
    const int pieces = cut.cta1 - cut.cta0 + 1;
    auto piece = [&](int i) { return p.slots + static_cast<int64_t>(2 * (cut.cta0 + i) + (i == 0)) * kTileSlot; };
    float top = -INFINITY, sum = 0.0f;
#pragma unroll 8
    for (int i = 0; i < pieces; ++i) top = max3_nan(top, __ldcg(piece(i) + kTileRows * kDim + r), top);
    float4 x[kFours] = {};
#pragma unroll (8 / kFours)
    for (int i = 0; i < pieces; ++i) {
        const float* at = piece(i);
        const float f = join_weight(__ldcg(at + kTileRows * kDim + r), top);
        sum += f * __ldcg(at + kTileRows * kDim + kTileRows + r);
#pragma unroll
        for (int j = 0; j < kFours; ++j) {
            const float4 y = __ldcg(reinterpret_cast<const float4*>(at) + ((r & ~31) + d4 + j) * 32 + (r & 31));
            x[j] = make_float4(x[j].x + f * y.x, x[j].y + f * y.y, x[j].z + f * y.z, x[j].w + f * y.w);
        }
    }
    const Seq s{cut.n, cut.kv, cut.q0};
    const int token = cut.token0 + tile_row / p.group, g = tile_row % p.group;
    int a, b;
    row_keys(p, s, token, a, b);
    const float inv = 1.0f / sum;
    const int64_t at = static_cast<int64_t>(cut.q0 + token) * p.heads * p.group + cut.head * p.group + g;
    uint2 y[kFours];
#pragma unroll
    for (int j = 0; j < kFours; ++j) {
        y[j] = make_uint2(pack2<T>(x[j].x * inv, x[j].y * inv), pack2<T>(x[j].z * inv, x[j].w * inv));
        if (b < a) y[j] = make_uint2(0, 0);
    }
    T* const out = static_cast<T*>(p.out) + at * kDim + d4 * 4;
    if constexpr (kFours == 1) {
        *reinterpret_cast<uint2*>(out) = y[0];
    } else {
#pragma unroll
        for (int j = 0; j < kFours; j += 2)
            reinterpret_cast<uint4*>(out)[j / 2] = make_uint4(y[j].x, y[j].y, y[j + 1].x, y[j + 1].y);
    }
    if (p.lse != nullptr && d4 == 0) p.lse[at] = b >= a ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_attend_join_kernel(const __grid_constant__ AttendParams p)
{
    wait_for_earlier_kernels();
    dependents_may_launch();
    const Cut cut = p.cuts[blockIdx.y];
    if (cut.cta1 == 0) return;
    const int sharers = cut.cta1 - cut.cta0, k = blockIdx.y - cut.cta0 - 1;
    const int fours = sharers >= 4 ? 1 : sharers >= 2 ? 2 : 4;
    const int part = blockIdx.x * (kJoinThreads / 32) + (threadIdx.x >> 5), d4 = part % 8 * 4 + k * fours;
    const int rows_per_tile = 128 / p.group * p.group, r = part / 8 * 32 + (threadIdx.x & 31);
    const int tile_row = r < 128 ? (r < rows_per_tile ? r : cut.rows) : (r - 128 < rows_per_tile ? rows_per_tile + r - 128 : cut.rows);
    if (k * fours >= 4 || tile_row >= cut.rows) return;
    if (fours == 4) join_values<T, 4>(p, cut, r, tile_row, d4);
    else if (fours == 2) join_values<T, 2>(p, cut, r, tile_row, d4);
    else join_values<T, 1>(p, cut, r, tile_row, d4);
}

// CTAs of a launch on the current device.
int attend_grid()
{
    static std::atomic<int> grids[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return kMaxGrid;
    std::atomic<int>& grid = grids[dev & 63];
    if ((n = grid.load(std::memory_order_relaxed)) > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return kMaxGrid;
    grid.store(n = n < kMaxGrid ? n : kMaxGrid, std::memory_order_relaxed);
    return n;
}

struct Device {
    bool rows_set[2] = {};
    bool tiles_set[2] = {};
};
std::mutex g_mu;
Device g_devices[64];

template <typename T>
int launch_rows(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttendParams& p, cudaStream_t stream)
{
    int dev = 0;
    cudaGetDevice(&dev);
    const int grid = attend_grid();
    {
        std::lock_guard<std::mutex> lock(g_mu);
        Device& d = g_devices[dev & 63];
        bool& set = d.rows_set[std::is_same<T, __half>::value];
        if (!set) {
            const cudaError_t e = cudaFuncSetAttribute(paged_attend_rows_kernel<T>,
                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem);
            if (e != cudaSuccess) return e;
            set = true;
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kRowsThreads);
    cfg.dynamicSmemBytes = kRowsSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    ProfileScope prof(kKernAttendRows, stream);
    return cudaLaunchKernelEx(&cfg, paged_attend_rows_kernel<T>, k_map, v_map, p);
}

template <typename T>
int launch_tiles(const CUtensorMap& q_map, const CUtensorMap& k_map, const CUtensorMap& v_map, const AttendParams& p,
                 cudaStream_t stream)
{
    int dev = 0;
    cudaGetDevice(&dev);
    const int grid = attend_grid();
    {
        std::lock_guard<std::mutex> lock(g_mu);
        Device& d = g_devices[dev & 63];
        bool& set = d.tiles_set[std::is_same<T, __half>::value];
        if (!set) {
            const cudaError_t e = cudaFuncSetAttribute(paged_attend_tiles_kernel<T>,
                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kTilesSmem);
            if (e != cudaSuccess) return e;
            set = true;
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kTileThreads);
    cfg.dynamicSmemBytes = kTilesSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    {
        ProfileScope prof(kKernAttendTiles, stream);
        const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_attend_tiles_kernel<T>, q_map, k_map, v_map, p);
        if (e != cudaSuccess) return e;
    }
    cfg.gridDim = dim3(kJoinBlocks, grid);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = 0;
    ProfileScope prof(kKernAttendJoin, stream);
    return cudaLaunchKernelEx(&cfg, paged_attend_join_kernel<T>, p);
}

}  // namespace

int launch_attend_tiles(const CUtensorMap& q_map, const CUtensorMap& k_map, const CUtensorMap& v_map,
                        const AttendParams& p, uint32_t dtype, cudaStream_t stream)
{
    return dtype == SECURE_INFER_FP16 ? launch_tiles<__half>(q_map, k_map, v_map, p, stream)
                                      : launch_tiles<__nv_bfloat16>(q_map, k_map, v_map, p, stream);
}

int launch_attend_rows(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttendParams& p, uint32_t dtype,
                       cudaStream_t stream)
{
    return dtype == SECURE_INFER_FP16 ? launch_rows<__half>(k_map, v_map, p, stream)
                                      : launch_rows<__nv_bfloat16>(k_map, v_map, p, stream);
}

uint64_t attend_workspace_bytes()
{
    return kSlotOffset + static_cast<uint64_t>(2 * attend_grid()) * (kTileSlot + kRowSlot) * sizeof(float);
}

void attend_workspace(void* workspace, AttendParams* p)
{
    p->status = static_cast<uint32_t*>(workspace);
    p->counters = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + kCounterOffset);
    p->cuts = reinterpret_cast<Cut*>(static_cast<char*>(workspace) + kCutOffset);
    p->slots = reinterpret_cast<float*>(static_cast<char*>(workspace) + kSlotOffset);
    p->row_slots = p->slots + static_cast<uint64_t>(2 * attend_grid()) * kTileSlot;
}

}  // namespace paged
}  // namespace sib
