// paged_cache.cu -- rotary positions with the way of new keys and values into
// their pages, and the copying, forking, reserving, freeing and compacting of
// pages.
#include "paged.cuh"
#include "gcm_kernels.cuh"

namespace sib {
namespace paged {
namespace {

// ------------------------------------------------------------------ append
//
// Pair i of a token's head turns by a = 2 pi pos f_i / 2^64, f_i = base^(-i/64)
// 2^64 / 2 pi: (x, y) -> (x cos a - y sin a, y cos a + x sin a).  The product
// pos f_i modulo 2^64 is the exact fraction of a turn, so the angle is as good
// at position 10^6 as at 1, where a 32-bit product pos f would have lost it.
// It cannot do without reading and writing each row once.  Eight lanes hold a row
// (eight pairs each, 16-byte accesses), a warp four rows at a time, and computes
// its lanes' eight angles once for all rows that it turns.  Measured: 6237 tokens
// of 28 query and 4 KV heads 23 us, 4.9 TB/s, where the copy rate would take 17.6
// (27 us before rows were loaded ahead of the angles).  Memory is not what bounds
// it: 1560 blocks are one and a half times what fits at 72 registers, and issue is
// half busy.  16 tokens of 32 and 8 heads: 3.7 us.
constexpr int kAppendThreads = 128;
// Twelve rows of a warp on their way at once: 23.0 us for the 6237 tokens; with 16, 20, 24 or 36 rows 26.7, 24.6, 27.1
// and 27.0 (fewer warps for their registers), with twelve in 64 registers of a thread instead of 72 26.5.
constexpr int kAppendBatch = 3;

__device__ __forceinline__ int find_seq(const int32_t* cu, int seqs, int token)
{
    // The last s with cu[s] <= token: 32 probes at a time.
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = seqs;   // cu[lo] <= token, and the answer lies in [lo, hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const uint32_t below = __ballot_sync(0xffffffffu, at < hi && cu[at] <= token);
        const int k = below == 0 ? 0 : 31 - __clz(below);
        lo += k * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

template <typename T>
__global__ void __launch_bounds__(kAppendThreads)
paged_append_kernel(const __grid_constant__ AppendParams p, int groups, int rows_per_warp)
{
    const int lane = threadIdx.x & 31, sub = lane & 7;
    const int64_t work = static_cast<int64_t>(blockIdx.x) * (kAppendThreads / 32) + (threadIdx.x >> 5);
    const int64_t token64 = work / groups;
    wait_for_earlier_kernels();
    dependents_may_launch();
    if (token64 >= p.tokens) return;
    const int token = static_cast<int>(token64), part = static_cast<int>(work % groups);
    const int rotated = p.q_heads + p.heads;
    const int row0 = part * rows_per_warp, row1 = min(row0 + rows_per_warp, rotated + p.heads);
    const int lo = p.interleaved ? sub * 16 : sub * 8, hi = p.interleaved ? sub * 16 + 8 : 64 + sub * 8;
    // Twelve rows are on their way before the token's place and angles are known.
    uint4 a[kAppendBatch], b[kAppendBatch];
    auto load = [&](int first) {
#pragma unroll
        for (int i = 0; i < kAppendBatch; ++i) {
            const int row = first + 4 * i + (lane >> 3);
            if (row >= row1) break;
            const T* src = row < p.q_heads ? static_cast<const T*>(p.q) + token * p.q_stride[0] + row * p.q_stride[1]
                           : row < rotated ? static_cast<const T*>(p.k) + token * p.k_in[0] + (row - p.q_heads) * p.k_in[1]
                                           : static_cast<const T*>(p.v) + token * p.v_in[0] + (row - rotated) * p.v_in[1];
            a[i] = *reinterpret_cast<const uint4*>(src + lo);
            b[i] = *reinterpret_cast<const uint4*>(src + hi);
        }
    };
    load(row0);
    const int s = find_seq(p.cu, p.seqs, token);
    const int first = p.cu[s], end = min(p.cu[s + 1], p.tokens), kv = p.kv[s];
    const bool owned = token >= first && token < end;   // else the token is nobody's: q turns, nothing is written
    const int pos = kv - (end - first) + (token - first);
    int64_t k_at = -1, v_at = -1;
    if (owned && pos >= 0 && pos / kPage < p.width) {
        const int page = p.table[s * p.table_stride + pos / kPage];
        if (page >= 0 && page < p.pages) {
            k_at = page * p.k_stride[0] + (pos % kPage) * p.k_stride[1];
            v_at = page * p.v_stride[0] + (pos % kPage) * p.v_stride[1];
        }
    }
    float cs[8], sn[8];
    const bool turn = p.phase != nullptr && row0 < rotated;
    if (turn) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int pair = sub * 8 + i;
            const uint32_t axis = min(p.axis[pair], static_cast<uint32_t>(p.axes - 1));
            const int at = p.positions != nullptr ? p.positions[axis * p.position_stride + token] : pos;
            const uint64_t frac = static_cast<uint64_t>(static_cast<int64_t>(at)) * p.phase[pair];
            // Half turns in [-1, 1).
            sincospif(static_cast<float>(static_cast<int32_t>(frac >> 32)) * 0x1p-31f, &sn[i], &cs[i]);
        }
    }
    for (int batch = row0; batch < row1; batch += 4 * kAppendBatch) {
        if (batch > row0) load(batch);
#pragma unroll
        for (int i = 0; i < kAppendBatch; ++i) {
            const int row = batch + 4 * i + (lane >> 3);
            if (row >= row1) break;
            T* dst = nullptr;
            if (row < p.q_heads)
                dst = static_cast<T*>(p.q_out) + (static_cast<int64_t>(token) * p.q_heads + row) * kDim;
            else if (row < rotated)
                dst = k_at >= 0 ? static_cast<T*>(p.k_cache) + k_at + (row - p.q_heads) * p.k_stride[2] : nullptr;
            else
                dst = v_at >= 0 ? static_cast<T*>(p.v_cache) + v_at + (row - rotated) * p.v_stride[2] : nullptr;
            if (dst == nullptr) continue;
            if (turn && row < rotated) {
                uint32_t w[8] = {a[i].x, a[i].y, a[i].z, a[i].w, b[i].x, b[i].y, b[i].z, b[i].w};
                if (p.interleaved) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float2 u = unpack2<T>(w[j]);
                        w[j] = pack2<T>(u.x * cs[j] - u.y * sn[j], u.y * cs[j] + u.x * sn[j]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 u = unpack2<T>(w[j]), v = unpack2<T>(w[j + 4]);
                        w[j] = pack2<T>(u.x * cs[2 * j] - v.x * sn[2 * j], u.y * cs[2 * j + 1] - v.y * sn[2 * j + 1]);
                        w[j + 4] = pack2<T>(v.x * cs[2 * j] + u.x * sn[2 * j], v.y * cs[2 * j + 1] + u.y * sn[2 * j + 1]);
                    }
                }
                a[i] = make_uint4(w[0], w[1], w[2], w[3]);
                b[i] = make_uint4(w[4], w[5], w[6], w[7]);
            }
            *reinterpret_cast<uint4*>(dst + lo) = a[i];
            *reinterpret_cast<uint4*>(dst + hi) = b[i];
        }
    }
}

// --------------------------------------------------------------- page copy
//
// Bound by reading and writing every byte once: 16 KiB pieces, four 16-byte
// loads in flight per thread.  Measured: 32 pages of 16 MiB (32 layers of 8 heads)
// 165 us, 6.5 TB/s.
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;
constexpr int kCopyPiece = kCopyThreads * kCopyUnroll * 16;

__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(const __grid_constant__ CopyParams p)
{
    wait_for_earlier_kernels();
    const int n = p.count != nullptr ? min(*p.count, p.n) : p.n;
    const int pieces = static_cast<int>((p.page_bytes + kCopyPiece - 1) / kCopyPiece);
    const int64_t per_pair = static_cast<int64_t>(pieces) * p.tensors, total = per_pair * n;
    for (int64_t i = blockIdx.x; i < total; i += gridDim.x) {
        const int pair = static_cast<int>(i / per_pair), rest = static_cast<int>(i % per_pair);
        const int t = rest / pieces, piece = rest % pieces;
        const int src = p.src[pair], dst = p.dst[pair];
        if (src < 0 || src >= p.pages || dst < 0 || dst >= p.pages) continue;
        const char* from = static_cast<const char*>(p.t[t].base) + src * p.t[t].page_stride;
        char* to = static_cast<char*>(p.t[t].base) + dst * p.t[t].page_stride;
        uint4 x[kCopyUnroll];
#pragma unroll
        for (int j = 0; j < kCopyUnroll; ++j) {
            const int64_t at = static_cast<int64_t>(piece) * kCopyPiece + (j * kCopyThreads + threadIdx.x) * 16;
            if (at < p.page_bytes) x[j] = *reinterpret_cast<const uint4*>(from + at);
        }
#pragma unroll
        for (int j = 0; j < kCopyUnroll; ++j) {
            const int64_t at = static_cast<int64_t>(piece) * kCopyPiece + (j * kCopyThreads + threadIdx.x) * 16;
            if (at < p.page_bytes) *reinterpret_cast<uint4*>(to + at) = x[j];
        }
    }
}

// ------------------------------------------------------------------- tables
//
// The bookkeeping is integer work on some hundred KiB, bound by latency: one
// cluster of CTAs does an operation in one launch, its phases apart by cluster
// barriers.  Ranks come from prefix sums in page or request order, so pages
// are given and moved in one order whatever the timing; the only atomics are
// integer additions to the counts and a minimum over request numbers.  Measured:
// 300 of 512 sequences freed in a table of 256 columns and 20000 pages 7.9 us, one
// token reserved for each of 256 sequences (64 columns, 20000 pages) 7.7, of 1024
// 11.4.
constexpr int kMaxCluster = 8;
constexpr int kTableThreads = 1024;
// Entries up to which one CTA is faster than a cluster and its barriers.
constexpr int64_t kOneCta = 16384;

template <int kCluster>
__device__ __forceinline__ void cluster_barrier()
{
    if (kCluster == 1) {
        __syncthreads();
        return;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Sum of x over the threads before this one; `total`: over all.  sums: 33 ints.
__device__ __forceinline__ int block_prefix(int x, int* sums, int& total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int sum = x;
    for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += up;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = sum;
    __syncthreads();
    if (warp == 0) {
        const int own = sums[lane];
        int s = own;
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, s, d);
            if (lane >= d) s += up;
        }
        sums[lane] = s - own;
        if (lane == 31) sums[32] = s;
    }
    __syncthreads();
    total = sums[32];
    return sums[warp] + sum - x;
}

struct Scratch {
    int32_t *copies, *counts, *first, *second, *owner, *row_of, *place;
};

__host__ __device__ inline Scratch scratch_of(int32_t* s, uint32_t pages, uint32_t seqs)
{
    Scratch r;
    r.copies = s;                   // copies to make
    r.counts = s + 32;              // [3][kMaxCluster] per-CTA counts
    r.first = s + 64;               // [pages] free pages, or copy sources
    r.second = r.first + pages;     // [pages] copy destinations
    r.owner = r.second + pages;     // [seqs] first request that names the sequence
    r.row_of = r.owner + seqs;      // [seqs] request granted to the sequence, -1
    r.place = r.row_of + seqs;      // [n] pages given to earlier requests
    return r;
}

__device__ __forceinline__ int pages_of(int tokens, int width) { return min((max(tokens, 0) + kPage - 1) / kPage, width); }

template <int kOp, int kCluster>
__global__ void __launch_bounds__(kTableThreads, 1) page_tables_kernel(const __grid_constant__ TableParams p)
{
    __shared__ int sums[33];
    __shared__ int needs[kOp == kFork || kOp == kReserve ? kTableThreads + 1 : 1];
    wait_for_earlier_kernels();
    const int tid = threadIdx.x, cta = blockIdx.x, lane = tid & 31;
    const int all = cta * kTableThreads + tid, stride = kCluster * kTableThreads;
    const int pages = p.in.pages, seqs = p.in.seqs, width = p.in.width;
    const Scratch s = scratch_of(p.scratch, pages, seqs);
    const int slice = (pages + kCluster - 1) / kCluster, page0 = cta * slice, page1 = min(pages, page0 + slice);

    // Free pages (fork, reserve) or used ones (compact) of this CTA's slice; counts go over unless compacted.
    int found = 0;
    for (int i = page0 + tid; i < page1; i += kTableThreads) {
        const int r = p.in.refs[i];
        if (kOp != kCompact) p.out.refs[i] = r;
        found += kOp == kCompact ? r > 0 : r == 0;
    }
    if (kOp != kFree) {
        int total;
        block_prefix(found, sums, total);
        if (tid == 0) s.counts[cta] = total;
    }
    if (kOp != kCompact)
        for (int i = all; i < seqs; i += stride) s.owner[i] = INT32_MAX, s.row_of[i] = -1;
    cluster_barrier<kCluster>();

    if (kOp == kFork || kOp == kReserve) {
        const int32_t* named = kOp == kFork ? p.b : p.a;
        for (int i = all; i < p.n; i += stride)
            if (named[i] >= 0 && named[i] < seqs) atomicMin(&s.owner[named[i]], i);
        cluster_barrier<kCluster>();
        int free_before = 0, free_all = 0;
        for (int c = 0; c < kCluster; ++c) {
            const int k = __ldcg(&s.counts[c]);
            if (c < cta) free_before += k;
            free_all += k;
        }
        // Every CTA walks the requests, CTA 0 writes what it finds.  Where a block of them asks for more than is left one
        // thread goes through them, as a request that finds too few pages leaves them to the next: 1024 take it 13 us.
        int needed = 0;
        for (int i0 = 0; i0 < p.n; i0 += kTableThreads) {
            const int i = i0 + tid;
            bool ok = false;
            int need = 0, to = -1;
            if (i < p.n) {
                to = named[i];
                ok = to >= 0 && to < seqs && __ldcg(&s.owner[to]) == i;
                if (kOp == kFork) {
                    const int from = p.a[i];
                    ok = ok && from >= 0 && from < seqs && p.in.lens[to] == 0;
                    if (ok) {
                        const int len = max(p.in.lens[from], 0);
                        ok = len <= width * kPage;
                        need = ok && len % kPage != 0;
                    }
                } else if (ok) {
                    const int old = max(p.in.lens[to], 0), now = p.b[i], used = pages_of(old, width);
                    ok = old <= width * kPage && now >= old && now <= width * kPage;
                    if (ok && now > old && old % kPage != 0) {
                        const int last = p.in.block_table[static_cast<int64_t>(to) * width + used - 1];
                        ok = last >= 0 && last < pages && p.in.refs[last] == 1;
                    }
                    need = ok ? pages_of(now, width) - used : 0;
                }
            }
            int total;
            int place = block_prefix(need, sums, total);
            // (Sums of needs this large might pass 32 bits.)
            if (__syncthreads_or(need > 1 << 20) || total > free_all - needed) {
                needs[tid] = need;
                __syncthreads();
                if (tid == 0) {
                    const int left = free_all - needed;
                    int taken = 0;
                    for (int k = 0; k < min(kTableThreads, p.n - i0); ++k) {
                        const int want = needs[k];
                        const bool fits = want <= left - taken;
                        needs[k] = fits ? taken : -1;
                        taken += fits ? want : 0;
                    }
                    needs[kTableThreads] = taken;
                }
                __syncthreads();
                place = needs[tid];
                ok = ok && place >= 0;
                total = needs[kTableThreads];
            }
            place += needed;
            needed += total;
            if (cta == 0 && i < p.n) {
                p.granted[i] = ok;
                s.place[i] = place;
                if (ok) s.row_of[to] = i;
            }
        }
        // The lowest free pages, in order.
        int rank0 = free_before;
        for (int i0 = page0; i0 < page1 && rank0 < needed; i0 += kTableThreads) {
            const int i = i0 + tid;
            const int is_free = i < page1 && p.in.refs[i] == 0;
            int total;
            const int rank = rank0 + block_prefix(is_free, sums, total);
            rank0 += total;
            if (is_free && rank < needed) {
                if (kOp == kFork) s.second[rank] = i;
                else s.first[rank] = i;
            }
        }
        if (kOp == kFork && cta == 0 && tid == 0) *s.copies = needed;
        cluster_barrier<kCluster>();
    }
    if (kOp == kFree) {
        for (int i = all; i < p.n; i += stride)
            if (p.a[i] >= 0 && p.a[i] < seqs) s.row_of[p.a[i]] = i;
        cluster_barrier<kCluster>();
    }
    if (kOp == kCompact) {
        int live = 0;
        for (int c = 0; c < kCluster; ++c) live += __ldcg(&s.counts[c]);
        int holes = 0, movers = 0;
        for (int i = page0 + tid; i < page1; i += kTableThreads) {
            const int r = p.in.refs[i];
            holes += r <= 0 && i < live;
            movers += r > 0 && i >= live;
            p.out.refs[i] = i < live ? r : 0;
            p.moved[i] = r > 0 ? i : -1;
        }
        int total;
        block_prefix(holes, sums, total);
        if (tid == 0) s.counts[kCluster + cta] = total;
        block_prefix(movers, sums, total);
        if (tid == 0) s.counts[2 * kCluster + cta] = total;
        cluster_barrier<kCluster>();
        int hole0 = 0, mover0 = 0, moves = 0;
        for (int c = 0; c < kCluster; ++c) {
            if (c < cta) hole0 += __ldcg(&s.counts[kCluster + c]);
            if (c < cta) mover0 += __ldcg(&s.counts[2 * kCluster + c]);
            moves += __ldcg(&s.counts[2 * kCluster + c]);
        }
        for (int i0 = page0; i0 < page1; i0 += kTableThreads) {
            const int i = i0 + tid;
            const int r = i < page1 ? p.in.refs[i] : 0;
            const int hole = i < page1 && r <= 0 && i < live, mover = i < page1 && r > 0 && i >= live;
            int n_holes, n_movers;
            const int h = hole0 + block_prefix(hole, sums, n_holes), m = mover0 + block_prefix(mover, sums, n_movers);
            if (hole) s.second[h] = i;
            if (mover) s.first[m] = i;
            hole0 += n_holes;
            mover0 += n_movers;
        }
        cluster_barrier<kCluster>();
        for (int k = all; k < moves; k += stride) {
            const int from = __ldcg(&s.first[k]), to = __ldcg(&s.second[k]);
            p.moved[from] = to;
            p.out.refs[to] = p.in.refs[from];
        }
        if (cta == 0 && tid == 0) {
            *s.copies = moves;
            *p.live = live;
        }
        cluster_barrier<kCluster>();
    }

    // The rows, a warp each.
    dependents_may_launch();
    for (int r = all >> 5; r < seqs; r += stride >> 5) {
        const int32_t* in = p.in.block_table + static_cast<int64_t>(r) * width;
        int32_t* out = p.out.block_table + static_cast<int64_t>(r) * width;
        const int len = max(p.in.lens[r], 0), used = pages_of(len, width);
        int now = len;
        if (kOp == kCompact) {
            for (int c = lane; c < width; c += 32) {
                const int page = in[c];
                out[c] = c < used && page >= 0 && page < pages ? __ldcg(&p.moved[page]) : -1;
            }
        } else {
            const int i = __ldcg(&s.row_of[r]);
            if (i < 0) {
                for (int c = lane; c < width; c += 32) out[c] = in[c];
                now = p.in.lens[r];
            } else if (kOp == kFree) {
                now = 0;
                for (int c = lane; c < width; c += 32) {
                    const int page = in[c];
                    if (c < used && page >= 0 && page < pages) atomicSub(&p.out.refs[page], 1);
                    out[c] = -1;
                }
            } else if (kOp == kReserve) {
                now = p.b[i];
                const int place = __ldcg(&s.place[i]), grown = pages_of(now, width);
                for (int c = lane; c < width; c += 32) {
                    int page = in[c];
                    if (c >= used && c < grown) {
                        page = __ldcg(&s.first[place + c - used]);
                        p.out.refs[page] = 1;
                    }
                    out[c] = page;
                }
            } else {
                const int from = p.a[i], place = __ldcg(&s.place[i]);
                now = max(p.in.lens[from], 0);
                const int full = now / kPage;
                for (int c = lane; c < width; c += 32) {
                    int page = -1;
                    if (c < full) {
                        page = p.in.block_table[static_cast<int64_t>(from) * width + c];
                        if (page >= 0 && page < pages) atomicAdd(&p.out.refs[page], 1);
                    } else if (c == full && now % kPage != 0) {
                        page = __ldcg(&s.second[place]);
                        p.out.refs[page] = 1;
                        s.first[place] = p.in.block_table[static_cast<int64_t>(from) * width + c];
                    }
                    out[c] = page;
                }
            }
        }
        if (lane == 0) p.out.lens[r] = now;
    }
}

template <int kOp, int kCluster>
cudaError_t launch_op_on(const TableParams& p, cudaStream_t stream)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kCluster);
    cfg.blockDim = dim3(kTableThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kCluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = kCluster > 1 ? 2 : 1;
    ProfileScope prof(kKernTables, stream);
    return cudaLaunchKernelEx(&cfg, page_tables_kernel<kOp, kCluster>, p);
}

template <int kOp>
cudaError_t launch_op(const TableParams& p, cudaStream_t stream)
{
    const int64_t entries = static_cast<int64_t>(p.in.seqs) * p.in.width + p.in.pages;
    return entries <= kOneCta ? launch_op_on<kOp, 1>(p, stream) : launch_op_on<kOp, kMaxCluster>(p, stream);
}

int sm_count()
{
    static int counts[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (counts[dev & 63] == 0) {
        int n = 0;
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        counts[dev & 63] = n;
    }
    return counts[dev & 63];
}

}  // namespace

int launch_append(const AppendParams& p, uint32_t dtype, cudaStream_t stream)
{
    if (p.tokens == 0) return cudaSuccess;
    // A warp turns as many rows of a token as leave about 16 warps per SM: all of them in a large chunk, so its
    // angles are computed once, four in a small one, where the rows side by side are what shortens the call.
    const int rows = p.q_heads + 2 * p.heads;
    const int64_t warps = 16 * static_cast<int64_t>(sm_count());
    int64_t per = (static_cast<int64_t>(p.tokens) * rows + warps - 1) / warps;
    per = (per + 3) / 4 * 4;
    if (per > rows) per = rows;
    const int groups = static_cast<int>((rows + per - 1) / per);
    const int64_t blocks = (static_cast<int64_t>(p.tokens) * groups + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
    if (blocks > INT32_MAX) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<uint32_t>(blocks));
    cfg.blockDim = dim3(kAppendThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    ProfileScope prof(kKernAppend, stream);
    if (dtype == SECURE_INFER_FP16)
        return cudaLaunchKernelEx(&cfg, paged_append_kernel<__half>, p, groups, static_cast<int>(per));
    return cudaLaunchKernelEx(&cfg, paged_append_kernel<__nv_bfloat16>, p, groups, static_cast<int>(per));
}

int launch_page_copy(const secure_infer_page_tensor* tensors, uint32_t n_tensors, uint64_t page_bytes, uint32_t pages,
                     const int32_t* src, const int32_t* dst, const int32_t* count, uint32_t n, cudaStream_t stream)
{
    if (n == 0) return cudaSuccess;
    for (uint32_t t0 = 0; t0 < n_tensors; t0 += kCopyTensors) {
        CopyParams p;
        p.src = src;
        p.dst = dst;
        p.count = count;
        p.n = static_cast<int32_t>(n);
        p.pages = static_cast<int32_t>(pages);
        p.tensors = static_cast<int32_t>(n_tensors - t0 < kCopyTensors ? n_tensors - t0 : kCopyTensors);
        p.page_bytes = static_cast<int64_t>(page_bytes);
        for (int i = 0; i < p.tensors; ++i) p.t[i] = tensors[t0 + i];
        const int64_t pieces = static_cast<int64_t>((page_bytes + kCopyPiece - 1) / kCopyPiece) * p.tensors * n;
        // Many more blocks than fit at once, so that SMs with a shorter way to memory take more pieces: 1.07 GB in
        // 179 us with the 8 blocks per SM that fit, 165 with 64; more cost a list shorter than its bound too much.
        const int64_t cap = 64 * static_cast<int64_t>(sm_count());
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(static_cast<uint32_t>(pieces < cap ? pieces : cap));
        cfg.blockDim = dim3(kCopyThreads);
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        ProfileScope prof(kKernPageCopy, stream);
        const cudaError_t e = cudaLaunchKernelEx(&cfg, page_copy_kernel, p);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

uint64_t table_scratch_ints(uint32_t seqs, uint32_t pages, uint32_t n)
{
    return 64 + 2 * static_cast<uint64_t>(pages) + 2 * static_cast<uint64_t>(seqs) + n;
}

CopyList table_copy_list(int32_t* scratch, uint32_t pages)
{
    const Scratch s = scratch_of(scratch, pages, 0);
    return CopyList{s.copies, s.first, s.second};
}

int launch_tables(TableOp op, const TableParams& p, cudaStream_t stream)
{
    switch (op) {
        case kFork: return launch_op<kFork>(p, stream);
        case kReserve: return launch_op<kReserve>(p, stream);
        case kFree: return launch_op<kFree>(p, stream);
        default: return launch_op<kCompact>(p, stream);
    }
}

}  // namespace paged
}  // namespace sib
