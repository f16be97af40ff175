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

#include <mutex>

namespace sib {
namespace paged {
namespace {

// Workspace: counters, the status word, then partial results.
constexpr int kMaxGrid = 256;
constexpr uint64_t kSlotOffset = 4096;

// ---------------------------------------------------------------- few rows
//
// Single tokens and short drafts: at most 16 * kTiles rows per KV head and
// tile, bound by reading K and V once.  One CTA per SM; a producer warp keeps
// three pages (64 KiB each, K and V) in flight by TMA; each of eight warps takes
// 16 rows and a slice of each page's keys: scores by m16n8k16 with the rows as
// M, their own running maximum and sum, and the values' product, so no warp
// waits for another inside the loop.  The results join in shared memory at the tile's end,
// and a tile cut over several CTAs is joined by the last of them to finish, in
// the order of the cuts, so results do not depend on the order of arrival.
constexpr int kRowsWarps = 8;
constexpr int kRowsThreads = 32 * (kRowsWarps + 1);
constexpr int kRowsStages = 3;
constexpr int kQuarter = 32;                              // tokens of one TMA box
constexpr uint32_t kQuarterBytes = kQuarter * kDim * 2;   // [2 halves][32 tokens][64 values]
constexpr uint32_t kPageTile = 4 * kQuarterBytes;         // K or V of one page and head
constexpr int kMaxRowTiles = 4;
constexpr uint32_t kJoinBytes = kRowsWarps * 8 * 64 * 4;  // 8 rows x 64 columns of every warp
constexpr uint32_t kRowsSmem = 1024 + kRowsStages * 2 * kPageTile + kMaxRowTiles * 16 * 256 + kJoinBytes +
                               2 * kRowsWarps * 16 * 4;
// Partial result of a CTA: [rows][128] sums, [rows] maxima, [rows] sums.
constexpr int kRowsMinUnits = 1;
constexpr int kRowSlot = kMaxRowTiles * 16 * (kDim + 2);

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

// Barrier of the eight computing warps.
__device__ __forceinline__ void rows_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kRowsWarps) : "memory"); }

template <typename T, int kTiles>
__global__ void __launch_bounds__(kRowsThreads, 1)
paged_attend_rows_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                         const __grid_constant__ AttendParams p)
{
    constexpr int kRows = 16 * kTiles;            // eight warps: kTiles times 16 rows, kSlices slices of a page's keys
    constexpr int kSlices = kRowsWarps / kTiles;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[3 * kRowsStages];   // K full, V full, empty
    __shared__ Share share;
    __shared__ int64_t warp_sums[kRowsThreads / 32];
    __shared__ volatile int stop;   // a wait ran out
    __shared__ int irregular, last_piece, give_up;

    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t k_smem = smem_addr(base), v_smem = k_smem + kRowsStages * kPageTile;
    const uint32_t q_smem = v_smem + kRowsStages * kPageTile;
    uint8_t* q_bytes = base + 2 * kRowsStages * kPageTile;
    float* join = reinterpret_cast<float*>(q_bytes + kMaxRowTiles * 16 * 256);
    float* join_m = join + kJoinBytes / 4;
    float* join_l = join_m + kRowsWarps * 16;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row_tile = warp / kSlices;
    auto k_full = [&](int s) { return smem_addr(&bars[s]); };
    auto v_full = [&](int s) { return smem_addr(&bars[kRowsStages + s]); };
    auto empty = [&](int s) { return smem_addr(&bars[2 * kRowsStages + s]); };
    if (tid == 0) {
        for (int s = 0; s < kRowsStages; ++s) {
            barrier_init(k_full(s), 1);
            barrier_init(v_full(s), 1);
            barrier_init(empty(s), kRowsWarps);
        }
        stop = 0;
        irregular = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
    }
    wait_for_earlier_kernels();
    find_share<kRowsThreads>(p, kRows, kRowsMinUnits, &share, warp_sums);
    dependents_may_launch();
    Walk w = start_walk(p, kRows, share);

    if (warp == kRowsWarps) {
        // Producer: the quarters of each page that hold keys any row sees.
        int64_t unit = 0;
        while (w.left > 0 && !stop) {
            const int pages = static_cast<int>(min(w.left, static_cast<int64_t>(w.span.pages - w.page)));
            const int32_t* row = p.table + w.s * p.table_stride + w.span.first + w.page;
            for (int i0 = 0; i0 < pages; i0 += 32) {
                const int id = i0 + lane < pages && w.span.hi > 0 ? row[i0 + lane] : -1;
                for (int i = i0; i < min(pages, i0 + 32); ++i, ++unit) {
                    const int page = __shfl_sync(0xffffffffu, id, i - i0);
                    const int stage = static_cast<int>(unit % kRowsStages);
                    const uint32_t turn = static_cast<uint32_t>(unit / kRowsStages);
                    if (lane != 0 || stop || (turn > 0 && !barrier_wait(empty(stage), (turn - 1) & 1, &stop))) continue;
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
            w.left -= pages;
            if (w.left > 0) w.next_tile(p);
        }
        // Copies still in flight land before the CTA's shared memory goes away.
        if (lane == 0) {
            for (int64_t u = max(int64_t(0), unit - kRowsStages); u < unit; ++u) {
                barrier_wait(k_full(u % kRowsStages), static_cast<uint32_t>(u / kRowsStages) & 1, &stop);
                barrier_wait(v_full(u % kRowsStages), static_cast<uint32_t>(u / kRowsStages) & 1, &stop);
            }
            if (stop) atomicOr(p.status, 1u);
        }
        return;
    }

    int64_t unit = 0;
    while (w.left > 0) {
        const int pages = static_cast<int>(min(w.left, static_cast<int64_t>(w.span.pages - w.page)));
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
        rows_sync();

        int lo[2], hi[2];   // keys that this thread's rows see
        int all_lo, all_hi; // keys that every row of the tile sees
        {
            int unused;
            row_keys(p, w.q, w.last_token, all_lo, unused);
            row_keys(p, w.q, w.first_token, unused, all_hi);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = row_tile * 16 + h * 8 + (lane >> 2);
            row_keys(p, w.q, min(w.last_token, (r0 + r) / p.group), lo[h], hi[h]);
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[16][4];
#pragma unroll
        for (int d = 0; d < 16; ++d)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[d][c] = 0.0f;
        const bool idle = row_tile * 16 >= w.rows;   // no row of this warp's sixteen is used

        for (int i = 0; i < pages; ++i, ++unit) {
            const int stage = static_cast<int>(unit % kRowsStages);
            const uint32_t parity = static_cast<uint32_t>(unit / kRowsStages) & 1;
            const int page_key = (w.span.first + w.page + i) * kPage;
            if (!barrier_wait(k_full(stage), parity, &stop) || !barrier_wait(v_full(stage), parity, &stop)) break;
#pragma unroll
            for (int sub = 0; sub < kTiles; ++sub) {
                const int slot16 = (warp % kSlices) * kTiles + sub, key0 = page_key + slot16 * 16;
                if (idle || key0 >= w.span.hi || key0 + 16 <= w.span.lo) continue;
                const uint32_t slice = stage * kPageTile + (slot16 >> 1) * kQuarterBytes + (slot16 & 1) * 16 * 128;
                const bool whole = key0 >= all_lo && key0 + 15 <= all_hi;
                float s[2][4] = {};
#pragma unroll
                for (int d = 0; d < 8; ++d) {   // 16 values of the head at a time
                    uint32_t a[4], b[4];
                    const int key = (lane & 7) + ((lane >> 4) << 3), chunk = (d & 3) * 2 + ((lane >> 3) & 1);
                    ldmatrix4(b, k_smem + slice + (d >> 2) * (kQuarterBytes / 2) + key * 128 + ((chunk ^ (key & 7)) << 4));
                    const int r = row_tile * 16 + (lane & 15), piece = d * 2 + (lane >> 4);
                    ldmatrix4(a, q_smem + r * 256 + ((piece ^ (r & 7)) << 4));
                    mma16816<T>(s[0], a, b[0], b[1]);
                    mma16816<T>(s[1], a, b[2], b[3]);
                }
                float top[2] = {m[0], m[1]};
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float x = s[n][c] * p.scale_log2;
                        if (!whole) {
                            const int key = key0 + n * 8 + (lane & 3) * 2 + (c & 1);
                            if (key < lo[c >> 1] || key > hi[c >> 1]) x = -INFINITY;
                        }
                        s[n][c] = x;
                        top[c >> 1] = fmaxf(top[c >> 1], x);
                    }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                }
                if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float f = m[h] == top[h] ? 1.0f : exp2_approx(m[h] - top[h]);
                        m[h] = top[h];
                        l[h] *= f;
#pragma unroll
                        for (int d = 0; d < 16; ++d) {
                            o[d][2 * h] *= f;
                            o[d][2 * h + 1] *= f;
                        }
                    }
                }
                const float base0 = top[0] == -INFINITY ? 0.0f : top[0], base1 = top[1] == -INFINITY ? 0.0f : top[1];
                uint32_t weight[4];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float e0 = exp2_approx(s[n][0] - base0), e1 = exp2_approx(s[n][1] - base0);
                    const float e2 = exp2_approx(s[n][2] - base1), e3 = exp2_approx(s[n][3] - base1);
                    l[0] += e0 + e1;
                    l[1] += e2 + e3;
                    // Weights are rounded to the cache's type for the product; their sum is not.
                    weight[2 * n] = pack2<T>(e0, e1);
                    weight[2 * n + 1] = pack2<T>(e2, e3);
                }
                uint32_t keep[2] = {0, 0};   // values of keys that some row sees: this lane's keys 2t, 2t + 1 and 8 more
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = key0 + (j >> 1) * 8 + (lane & 3) * 2 + (j & 1);
                    if (key >= w.span.lo && key < w.span.hi) keep[j >> 1] |= (j & 1) ? 0xffff0000u : 0x0000ffffu;
                }
                bool odd = false;
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    uint32_t b[4];
                    const int key = lane & 15, chunk = (d & 3) * 2 + (lane >> 4);
                    ldmatrix4_trans(b, v_smem + slice + (d >> 2) * (kQuarterBytes / 2) + key * 128 +
                                           ((chunk ^ (key & 7)) << 4));
                    if (!whole) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            b[j] &= keep[j & 1];
                            odd |= nonfinite2<T>(b[j]);
                        }
                    }
                    mma16816<T>(o[2 * d], weight, b[0], b[1]);
                    mma16816<T>(o[2 * d + 1], weight, b[2], b[3]);
                }
                if (odd && w.first_token != w.last_token) irregular = 1;
            }
            __syncwarp();
            if (lane == 0) barrier_arrive(empty(stage));
        }

        // Join the warps' results.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if ((lane & 3) == 0) {
                join_m[warp * 16 + h * 8 + (lane >> 2)] = m[h];
                join_l[warp * 16 + h * 8 + (lane >> 2)] = l[h];
            }
        }
        if (tid == 0) give_up = stop;
        rows_sync();
        if (give_up) break;
        const int64_t tile_end = w.tile_unit + w.span.pages;
        const int cta0 = static_cast<int>(w.tile_unit / share.per), cta1 = static_cast<int>((tile_end - 1) / share.per);
        const bool split = cta1 > cta0;
        float* slot = p.slots + static_cast<int64_t>(2 * blockIdx.x + (static_cast<int>(blockIdx.x) == cta0)) * kRowSlot;
        const bool by_definition = irregular != 0;

        auto emit2 = [&](int r, int col, float2 x, float mm, float ll) {
            if (split) {
                *reinterpret_cast<float2*>(slot + r * kDim + col) = x;
                if (col == 0) {
                    slot[kRows * kDim + r] = mm;
                    slot[kRows * kDim + kRows + r] = ll;
                }
                return;
            }
            const int token = (r0 + r) / p.group, g = (r0 + r) % p.group;
            int a, b;
            row_keys(p, w.q, token, a, b);
            const float inv = 1.0f / ll;
            const int64_t at = static_cast<int64_t>(w.q.q0 + token) * p.heads * p.group + w.head * p.group + g;
            *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + at * kDim + col) =
                b >= a ? pack2<T>(x.x * inv, x.y * inv) : 0u;
            if (p.lse != nullptr && col == 0)
                p.lse[at] = b >= a ? (mm + log2f(ll)) * 0.6931471805599453f : -INFINITY;
        };

        if (!by_definition) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h * 8 >= w.rows) continue;   // the same for all threads
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int d = 0; d < 8; ++d)
                        *reinterpret_cast<float2*>(join + warp * 512 + (lane >> 2) * 64 + d * 8 + (lane & 3) * 2) =
                            make_float2(o[half * 8 + d][2 * h], o[half * 8 + d][2 * h + 1]);
                    rows_sync();
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) {
                        const int r = t * 16 + h * 8 + warp;
                        if (r >= w.rows) continue;
                        float top = -INFINITY;
#pragma unroll
                        for (int i = t * kSlices; i < (t + 1) * kSlices; ++i)
                            top = fmaxf(top, join_m[i * 16 + h * 8 + warp]);
                        float2 x = make_float2(0.0f, 0.0f);
                        float sum = 0.0f;
#pragma unroll
                        for (int i = t * kSlices; i < (t + 1) * kSlices; ++i) {
                            const float f = join_weight(join_m[i * 16 + h * 8 + warp], top);
                            const float2 y = *reinterpret_cast<const float2*>(join + i * 512 + warp * 64 + lane * 2);
                            sum += f * join_l[i * 16 + h * 8 + warp];
                            x.x += f * y.x;
                            x.y += f * y.y;
                        }
                        emit2(r, half * 64 + lane * 2, x, top, sum);
                    }
                    rows_sync();
                }
            }
        } else {
            const int ka = (w.span.first + w.page) * kPage, kb = ka + pages * kPage;
            for (int r = warp; r < w.rows; r += kRowsWarps) {
                const int token = (r0 + r) / p.group, g = (r0 + r) % p.group;
                int a, b;
                row_keys(p, w.q, token, a, b);
                float mm, ll;
                float4 x;
                row_by_definition<T>(p, static_cast<const T*>(p.q) + (w.q.q0 + token) * p.q_token +
                                            (w.head * p.group + g) * p.q_head,
                                     p.table + w.s * p.table_stride, w.head, max(a, ka), min(b + 1, kb), mm, ll, x);
                emit2(r, lane * 4, make_float2(x.x, x.y), mm, ll);
                emit2(r, lane * 4 + 2, make_float2(x.z, x.w), mm, ll);
            }
        }

        if (split) {
            // The last CTA of the tile joins its pieces.
            __threadfence();
            rows_sync();
            const int pieces = cta1 - cta0 + 1;
            if (tid == 0) last_piece = atomicInc(&p.counters[cta0], pieces - 1) == static_cast<uint32_t>(pieces - 1);
            rows_sync();
            if (last_piece) {
                __threadfence();
                auto piece = [&](int i) {
                    return p.slots + static_cast<int64_t>(2 * (cta0 + i) + (i == 0)) * kRowSlot;
                };
                for (int r = warp; r < w.rows; r += kRowsWarps) {
                    float top = -INFINITY;
                    for (int i = lane; i < pieces; i += 32) top = fmaxf(top, __ldcg(piece(i) + kRows * kDim + r));
                    for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    float sum = 0.0f;
#pragma unroll 4
                    for (int i = 0; i < pieces; ++i) {
                        const float* src = piece(i);
                        const float f = join_weight(__ldcg(src + kRows * kDim + r), top);
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(src + r * kDim + lane * 4));
                        sum += f * __ldcg(src + kRows * kDim + kRows + r);
                        x.x += f * y.x;
                        x.y += f * y.y;
                        x.z += f * y.z;
                        x.w += f * y.w;
                    }
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
        }
        if (by_definition) {
            rows_sync();
            if (tid == 0) irregular = 0;
        }
        rows_sync();
        w.left -= pages;
        if (w.left > 0) w.next_tile(p);
    }
}

struct Device {
    int sms = 0;
    bool rows_set[2][kMaxRowTiles] = {};
};
std::mutex g_mu;
Device g_devices[64];

template <typename T, int kTiles>
int launch_rows(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttendParams& p, cudaStream_t stream)
{
    int dev = 0;
    cudaGetDevice(&dev);
    int sms;
    {
        std::lock_guard<std::mutex> lock(g_mu);
        Device& d = g_devices[dev & 63];
        if (d.sms == 0) cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev);
        bool& set = d.rows_set[std::is_same<T, __half>::value][kTiles - 1];
        if (!set) {
            const cudaError_t e = cudaFuncSetAttribute(paged_attend_rows_kernel<T, kTiles>,
                                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem);
            if (e != cudaSuccess) return e;
            set = true;
        }
        sms = d.sms;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(sms < kMaxGrid ? sms : kMaxGrid);
    cfg.blockDim = dim3(kRowsThreads);
    cfg.dynamicSmemBytes = kRowsSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    ProfileScope prof(kKernAttendRows, stream);
    return cudaLaunchKernelEx(&cfg, paged_attend_rows_kernel<T, kTiles>, k_map, v_map, p);
}

}  // namespace

int launch_attend_rows(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttendParams& p, int m_tiles,
                       uint32_t dtype, cudaStream_t stream)
{
    if (dtype == SECURE_INFER_FP16)
        return m_tiles == 1   ? launch_rows<__half, 1>(k_map, v_map, p, stream)
               : m_tiles == 2 ? launch_rows<__half, 2>(k_map, v_map, p, stream)
                              : launch_rows<__half, 4>(k_map, v_map, p, stream);
    return m_tiles == 1   ? launch_rows<__nv_bfloat16, 1>(k_map, v_map, p, stream)
           : m_tiles == 2 ? launch_rows<__nv_bfloat16, 2>(k_map, v_map, p, stream)
                          : launch_rows<__nv_bfloat16, 4>(k_map, v_map, p, stream);
}

uint64_t attend_workspace_bytes()
{
    return kSlotOffset + static_cast<uint64_t>(2 * kMaxGrid) * kRowSlot * sizeof(float);
}

void attend_workspace(void* workspace, AttendParams* p)
{
    p->counters = static_cast<uint32_t*>(workspace);
    p->status = p->counters + kMaxGrid;
    p->slots = reinterpret_cast<float*>(static_cast<char*>(workspace) + kSlotOffset);
}

}  // namespace paged
}  // namespace sib
