// paged.cuh -- what the kernels on the paged KV cache share: launch
// descriptors, the walk over attention's work, barriers and copies.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <type_traits>

#include "../../include/secure_infer_paged.h"

namespace sib {
namespace paged {

constexpr int kPage = 128;   // tokens of a page
constexpr int kDim = 128;    // values of a head

// What a CTA's last unit of a cut tile leaves for the join.
struct Cut {
    int32_t cta1, cta0, rows, token0, head;   // the last CTA and the first; cta1 = 0: no such tile
    int32_t n, kv, q0;
};

struct AttendParams {
    const void* q;
    int64_t q_token, q_head;        // strides, elements
    const void* k;
    const void* v;
    int64_t k_stride[3], v_stride[3];
    void* out;
    float* lse;                     // or null
    const int32_t* table;
    int64_t table_stride;
    const int32_t* cu;
    const int32_t* kv;
    int32_t width, seqs, tokens, pages;
    int32_t heads, group;           // KV heads, query heads of each
    int32_t rows_min, rows_max;     // sequences with rows_min <= rows <= rows_max are this launch's
    int32_t causal, window;
    float scale_log2;               // scale * log2(e): the softmax runs in powers of two
    uint32_t* status;               // not zero: a wait ran out, and calls give NaN until the host has read it
    uint32_t* counters;             // three of each CTA, zero between launches
    Cut* cuts;                      // [grid]
    float* slots;                   // [2 * grid] partial results of tiles
    float* row_slots;               // and of the kernel for few rows
    int32_t both;                   // the call has a launch for few rows, and then one for the others, on the same SMs
};

// Launchers (cudaError_t values).
int launch_attend_rows(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttendParams& p, uint32_t dtype,
                       cudaStream_t stream);
// q_map: boxes of [128 / group tokens][group heads][64 values].
int launch_attend_tiles(const CUtensorMap& q_map, const CUtensorMap& k_map, const CUtensorMap& v_map,
                        const AttendParams& p, uint32_t dtype, cudaStream_t stream);
uint64_t attend_workspace_bytes();
void attend_workspace(void* workspace, AttendParams* p);   // its counters, status word and slots

struct AppendParams {
    const void* q;
    const void* k;
    const void* v;
    int64_t q_stride[2], k_in[2], v_in[2];
    void* q_out;
    void* k_cache;
    void* v_cache;
    int64_t k_stride[3], v_stride[3];
    const int32_t* table;
    int64_t table_stride;
    const int32_t* cu;
    const int32_t* kv;
    const uint64_t* phase;
    const uint32_t* axis;
    const int32_t* positions;
    int64_t position_stride;
    int32_t width, seqs, tokens, pages, q_heads, heads, axes, interleaved;
};
int launch_append(const AppendParams& p, uint32_t dtype, cudaStream_t stream);

constexpr int kCopyTensors = 240;   // tensors of one copy launch, passed by value
struct CopyParams {
    const int32_t* src;
    const int32_t* dst;
    const int32_t* count;           // entries of src and dst, or null: n
    int32_t n, pages, tensors;
    int64_t page_bytes;
    secure_infer_page_tensor t[kCopyTensors];
};
int launch_page_copy(const secure_infer_page_tensor* tensors, uint32_t n_tensors, uint64_t page_bytes, uint32_t pages,
                     const int32_t* src, const int32_t* dst, const int32_t* count, uint32_t n, cudaStream_t stream);

enum TableOp : int32_t { kFork, kReserve, kFree, kCompact };
struct TableParams {
    secure_infer_tables in, out;
    const int32_t* a;               // fork: parents; reserve, free: sequences
    const int32_t* b;               // fork: children; reserve: new lengths
    int32_t* granted;
    int32_t* moved;
    int32_t* live;
    int32_t* scratch;
    int32_t n;
};
int launch_tables(TableOp op, const TableParams& p, cudaStream_t stream);
uint64_t table_scratch_ints(uint32_t seqs, uint32_t pages, uint32_t n);
// Where a table kernel leaves the page copies to make, in scratch.
struct CopyList {
    int32_t *count, *src, *dst;
};
CopyList table_copy_list(int32_t* scratch, uint32_t pages);

#ifdef __CUDACC__
// ------------------------------------------------------------ device helpers

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void dependents_may_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_earlier_kernels() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ bool barrier_done(uint32_t bar, uint32_t parity)
{
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return done != 0;
}

constexpr long long kWaitClocks = 1ll << 32;   // some seconds

// Waits for the phase of parity `parity`.  The wait is bounded: where nothing has
// happened for some seconds stop[0] is set and every wait of the CTA gives up, so
// a protocol error ends the kernel instead of hanging it; the rows of the CTA
// become NaN then.  stop[1] goes up while warps are at work that may take longer
// than that, and the others wait on.  Returns whether the phase completed: the
// lanes of a warp are together and read one barrier, one flag and one clock, so
// they get one answer.  (Votes on it took a chunk of 512 tokens 1.2 us.)
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, volatile int* stop)
{
    if (barrier_done(bar, parity)) return true;
    long long start = clock64();
    int work = -1;
    while (!barrier_done(bar, parity)) {
        if (*stop) return false;
        if (clock64() - start > kWaitClocks) {
            const int now = stop[1] & INT32_MAX;
            if (now == work) {
                *stop = 1;
                return false;
            }
            work = now;
            start = clock64();
        }
    }
    return true;
}

// For copies and products that have been issued: they write memory that the CTA
// gives back at its end, so it waits for them even after another wait ran out,
// with a limit of its own.
__device__ __forceinline__ void barrier_drain(uint32_t bar, uint32_t parity)
{
    const long long start = clock64();
    while (!barrier_done(bar, parity))
        if (clock64() - start > 2 * kWaitClocks) return;
}

__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, uint32_t bar, int token, int half,
                                              int head, int page)
{
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(0), "r"(token), "r"(half), "r"(head), "r"(page)
        : "memory");
}

__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t x);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t x)
{
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t x)
{
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

// Sums of products with zero: NaN in either half as soon as an infinity or a
// NaN was among the values.
template <typename T>
__device__ __forceinline__ uint32_t zero_sum(uint32_t sum, uint32_t x);
template <>
__device__ __forceinline__ uint32_t zero_sum<__nv_bfloat16>(uint32_t sum, uint32_t x)
{
    asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(x), "r"(0u));
    return sum;
}
template <>
__device__ __forceinline__ uint32_t zero_sum<__half>(uint32_t sum, uint32_t x)
{
    asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(x), "r"(0u));
    return sum;
}
template <typename T>
__device__ __forceinline__ bool zero_sum_odd(uint32_t sum)
{
    const float2 x = unpack2<T>(sum);
    return x.x != x.x || x.y != x.y;
}

// ------------------------------------------------- attention's work, in order
//
// A sequence's rows are (new token, query head of the group), flattened, so one
// KV head's K and V serve the whole group.  A tile is kRows of them over one KV
// head; its units are the pages that any of its rows sees (one empty unit if
// none).  All units of a launch in the order sequence, tile, head, page are cut
// into equal consecutive shares, one per CTA: every CTA gets the same work
// whatever the lengths, and a long axis is split where there are few rows.
// What a tile takes besides its pages (its queries, its end) counts as `cost`
// units more, before its pages.  Units are counted in 32 bits; the host refuses
// more.
struct Seq {
    int n, kv, q0;   // new tokens, all tokens, first new token
};

// `others`: the sequences of the call's other launch, else of this one.
__device__ __forceinline__ Seq load_seq(const AttendParams& p, int s, bool others = false)
{
    Seq r;
    // From L2, as all that may be read before this kernel has waited for the one before it.
    int a = __ldcg(p.cu + s), b = __ldcg(p.cu + s + 1);
    a = max(0, min(a, p.tokens));
    b = max(a, min(b, p.tokens));
    r.q0 = a;
    r.n = b - a;
    r.kv = max(0, min(__ldcg(p.kv + s), p.width * kPage));
    const int64_t rows = static_cast<int64_t>(r.n) * p.group;
    if ((rows < p.rows_min || rows > p.rows_max) != others) r.n = 0;
    return r;
}

struct Span {
    int first, pages;   // page range of a tile
    int lo, hi;         // keys that any row of it sees: [lo, hi)
};

__device__ __forceinline__ Span tile_span(const AttendParams& p, const Seq& s, int first_token, int last_token)
{
    Span r;
    r.hi = p.causal ? min(s.kv, s.kv - s.n + last_token + 1) : s.kv;
    r.lo = p.window ? max(0, s.kv - s.n + first_token - p.window + 1) : 0;
    if (r.hi <= r.lo) {
        r.lo = r.hi = r.first = 0;
        r.pages = 1;
    } else {
        r.first = r.lo / kPage;
        r.pages = (r.hi + kPage - 1) / kPage - r.first;
    }
    return r;
}

// A launch's units cut into consecutive shares of `per` or, for the first
// `more` CTAs, per + 1 units; `ctas` of the grid have one.
struct Share {
    int32_t per, more, ctas, total;
    int32_t begin, units;      // of this CTA
    int32_t seq, seq_unit;     // sequence of its first unit, and that sequence's first unit
    int32_t down;              // the status word when the kernel began
    Seq q;

    __device__ __forceinline__ int begin_of(int cta) const { return cta * per + min(cta, more); }
    __device__ __forceinline__ int owner(int unit) const
    {
        const int cut = more * (per + 1);
        return unit < cut ? unit / (per + 1) : more + (unit - cut) / per;
    }
};

struct Walk {
    int rows_per_tile, cost;
    int s, tile, tiles, head;
    Seq q;
    Span span;
    int page;                            // next unit of the tile: 0 .. span.pages
    int first_token, last_token, rows;   // of the tile
    int tile_unit;                       // number of the tile's first page
    int left;                            // units of this CTA not yet taken

    __device__ __forceinline__ int take() const { return min(left, span.pages - page); }
    __device__ __forceinline__ void set_tile(const AttendParams& p)
    {
        const int r0 = tile * rows_per_tile;
        rows = min(rows_per_tile, q.n * p.group - r0);
        first_token = r0 / p.group;
        last_token = (r0 + rows - 1) / p.group;
        span = tile_span(p, q, first_token, last_token);
    }
    // After `taken` units: the next head, tile or sequence.
    __device__ __forceinline__ void advance(const AttendParams& p, int taken)
    {
        left -= taken;
        if (left > 0) left -= cost;
        if (left <= 0) return;
        tile_unit += span.pages + cost;
        page = 0;
        if (++head < p.heads) return;
        head = 0;
        if (++tile < tiles) {
            set_tile(p);
            return;
        }
        tile = 0;
        do {
            if (++s >= p.seqs) {   // only if lengths changed under the kernel
                left = 0;
                return;
            }
            q = load_seq(p, s);
        } while (q.n == 0);
        tiles = (q.n * p.group + rows_per_tile - 1) / rows_per_tile;
        set_tile(p);
    }
};

// Pages and cost of a tile.
__device__ __forceinline__ int tile_units(const AttendParams& p, const Seq& s, int rows_per_tile, int cost, int tile)
{
    const int r = tile * rows_per_tile;
    return tile_span(p, s, r / p.group, (min(r + rows_per_tile, s.n * p.group) - 1) / p.group).pages + cost;
}

// Up to so many tiles of a sequence are counted by one thread, more by a warp:
// for a chunk of 4096 tokens of 4 rows a count took 4 us by one thread.
constexpr int kOwnTiles = 4;

// Units of every lane's sequence; `largest`: of a tile of theirs.  All lanes call it.
__device__ __forceinline__ int seq_units(const AttendParams& p, const Seq& s, int rows_per_tile, int cost, int& largest)
{
    const int lane = threadIdx.x & 31;
    const int tiles = (s.n * p.group + rows_per_tile - 1) / rows_per_tile;
    int units = 0;
    if (tiles <= kOwnTiles) {
        for (int t = 0; t < tiles; ++t) {
            const int u = tile_units(p, s, rows_per_tile, cost, t);
            units += u;
            largest = max(largest, u);
        }
    }
    for (uint32_t many = __ballot_sync(0xffffffffu, tiles > kOwnTiles); many != 0; many &= many - 1) {
        const int from = __ffs(many) - 1, n = __shfl_sync(0xffffffffu, tiles, from);
        const Seq q{__shfl_sync(0xffffffffu, s.n, from), __shfl_sync(0xffffffffu, s.kv, from), 0};
        int sum = 0, most = 0;
        for (int t = lane; t < n; t += 32) {
            const int u = tile_units(p, q, rows_per_tile, cost, t);
            sum += u;
            most = max(most, u);
        }
        sum = __reduce_add_sync(0xffffffffu, sum);
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == from) units = sum, largest = max(largest, most);
    }
    return units * p.heads;
}

// How one kind of launch cuts its tiles, and what a unit of it costs an SM.
struct Kind {
    int rows_per_tile, cost, whole;
    int time;     // of a unit, in any measure that both kinds share
    int of_16;    // sixteenths of the SMs beyond which it gets no faster
};

// All threads of the block take part; `warp_sums` holds three values per warp.
// Where no tile has more than `whole` units a CTA gets the largest one's:
// cutting it would cost more than the few pages that it would save.  Where the
// call has work of both kinds each gets SMs by the time that its units take:
// the first CTAs of a launch work and the others leave theirs to the other
// launch, so reading pages for few rows goes on beside the products of many: 333
// tokens after 2167 and 15 single tokens of up to 4000 take 53 us, 62 one kind
// after the other.
template <int kThreads>
__device__ __forceinline__ void find_share(const AttendParams& p, const Kind& kind, const Kind& other, Share* share,
                                           int32_t* warp_sums)
{
    const int rows_per_tile = kind.rows_per_tile, cost = kind.cost, whole = kind.whole;
    constexpr int kWarps = kThreads / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int down = tid == 0 ? static_cast<int>(__ldcg(p.status)) : 0;
    Share r;
    r.begin = r.total = 0;
    // The first pass sums the units, the second finds the sequence that holds this CTA's first; where every sequence
    // has a thread one pass does both.
    const bool one = p.seqs <= kThreads;
    for (int pass = one ? 1 : 0; pass < 2; ++pass) {
        int base = 0, largest = 0, others = 0;
        for (int s0 = 0; s0 < p.seqs; s0 += kThreads) {
            const int s = s0 + tid;
            Seq q{};
            int own_largest = 0, unused = 0, beside = 0;
            if (s < p.seqs) q = load_seq(p, s);
            if (p.both && (one || pass == 0)) {
                Seq o{};
                if (s < p.seqs) o = load_seq(p, s, true);
                beside = __reduce_add_sync(0xffffffffu, seq_units(p, o, other.rows_per_tile, other.cost, unused));
            }
            const int own = seq_units(p, q, rows_per_tile, cost, own_largest);
            int sum = own;
            for (int d = 1; d < 32; d <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += up;
            }
            own_largest = __reduce_max_sync(0xffffffffu, own_largest);
            if (lane == 31) {
                warp_sums[warp] = sum;
                warp_sums[kWarps + warp] = own_largest;
                warp_sums[2 * kWarps + warp] = beside;
            }
            __syncthreads();
            int before = base;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const int x = warp_sums[w];
                if (w < warp) before += x;
                base += x;
                largest = max(largest, warp_sums[kWarps + w]);
                others += warp_sums[2 * kWarps + w];
            }
            if (one || (pass == 0 && s0 + kThreads >= p.seqs)) {
                r.total = base;
                int grid = gridDim.x;
                if (base > 0 && others > 0 && grid > 1) {
                    const float mine = static_cast<float>(base) * kind.time, theirs = static_cast<float>(others) * other.time;
                    const int most = max(1, grid * kind.of_16 / 16), least = grid - max(1, grid * other.of_16 / 16);
                    grid = max(max(1, least), min(min(most, grid - 1), __float2int_rn(grid * (mine / (mine + theirs)))));
                }
                r.ctas = max(1, min(grid, largest <= whole ? base / max(1, largest) : base));
                r.per = base / r.ctas;
                r.more = base - r.per * r.ctas;
                const int c = blockIdx.x;
                r.begin = r.begin_of(c);
                r.units = c < r.ctas ? r.per + (c < r.more) : 0;
                if (tid == 0) {
                    r.seq = -1;
                    r.seq_unit = 0;
                    r.down = down;
                    *share = r;
                }
                __syncthreads();
            }
            if (pass == 1) {
                const int first = before + sum - own;
                if (r.units > 0 && own > 0 && r.begin >= first && r.begin < first + own) {
                    share->seq = s;
                    share->seq_unit = first;
                    share->q = q;
                }
            }
            __syncthreads();
        }
    }
}

// All lanes of a warp call it.
__device__ __forceinline__ Walk start_walk(const AttendParams& p, int rows_per_tile, int cost, const Share& share)
{
    Walk w;
    w.rows_per_tile = rows_per_tile;
    w.cost = cost;
    w.left = 0;
    if (share.seq < 0) return w;
    w.left = share.units;
    w.s = share.seq;
    w.q = share.q;
    w.tiles = (w.q.n * p.group + rows_per_tile - 1) / rows_per_tile;
    w.tile = 0;
    w.tile_unit = share.seq_unit;
    int skip = share.begin - share.seq_unit;
    // Of a sequence of many tiles, 32 at a time.
    for (bool past = w.tiles > kOwnTiles; past;) {
        const int lane = threadIdx.x & 31, t = w.tile + lane;
        int upto = t < w.tiles ? tile_units(p, w.q, rows_per_tile, cost, t) * p.heads : 0;
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += up;
        }
        const int whole = __popc(__ballot_sync(0xffffffffu, t < w.tiles && upto <= skip));
        if (whole > 0) {
            const int units = __shfl_sync(0xffffffffu, upto, whole - 1);
            skip -= units;
            w.tile_unit += units;
            w.tile += whole;
        }
        past = whole == 32;
    }
    w.set_tile(p);
    int units = w.span.pages + cost;
    while (skip >= units * p.heads) {
        skip -= units * p.heads;
        w.tile_unit += units * p.heads;
        ++w.tile;
        w.set_tile(p);
        units = w.span.pages + cost;
    }
    w.head = skip / units;
    skip -= w.head * units;
    w.tile_unit += w.head * units + cost;
    w.page = max(0, skip - cost);
    w.left = max(0, w.left - max(0, cost - skip));   // a share of nothing but cost has no page
    return w;
}

// Keys that row r of the tile sees: [lo, hi].
__device__ __forceinline__ void row_keys(const AttendParams& p, const Seq& s, int token, int& lo, int& hi)
{
    hi = p.causal ? min(s.kv, s.kv - s.n + token + 1) - 1 : s.kv - 1;
    lo = p.window ? max(0, s.kv - s.n + token - p.window + 1) : 0;
}

// One row over keys [a, b) by one warp, straight from the pages: lane l holds
// values 4l .. 4l+3.  Only rows of a tile in which some row must not see an
// infinite or NaN value that another one does see come here: in a matrix
// product zero times such a value would be NaN.  A key takes about 430
// clocks, the rows of a long piece longer than the other warps' waits last, so
// it counts its way in *work.
template <typename T>
__device__ __noinline__ void row_by_definition(const AttendParams& p, const T* q, const int32_t* table, int head, int a,
                                               int b, float& m, float& l, float4& o, volatile int* work)
{
    const int d = 4 * (threadIdx.x & 31);
    const uint2 qx = __ldcg(reinterpret_cast<const uint2*>(q + d));
    const float2 q0 = unpack2<T>(qx.x), q1 = unpack2<T>(qx.y);
    m = -INFINITY;
    l = 0.0f;
    o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int j = a; j < b; ++j) {
        if (((j - a) & 1023) == 0 && d == 0) atomicAdd(const_cast<int*>(work), 1);
        const int page = __ldcg(table + j / kPage);
        float2 k0 = {0, 0}, k1 = {0, 0}, v0 = {0, 0}, v1 = {0, 0};
        if (page >= 0 && page < p.pages) {
            const uint2 kx = __ldcg(reinterpret_cast<const uint2*>(static_cast<const T*>(p.k) + page * p.k_stride[0] +
                                                                   (j % kPage) * p.k_stride[1] + head * p.k_stride[2] + d));
            const uint2 vx = __ldcg(reinterpret_cast<const uint2*>(static_cast<const T*>(p.v) + page * p.v_stride[0] +
                                                                   (j % kPage) * p.v_stride[1] + head * p.v_stride[2] + d));
            k0 = unpack2<T>(kx.x), k1 = unpack2<T>(kx.y), v0 = unpack2<T>(vx.x), v1 = unpack2<T>(vx.y);
        }
        float x = q0.x * k0.x + q0.y * k0.y + q1.x * k1.x + q1.y * k1.y;
        for (int s = 16; s; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
        x *= p.scale_log2;
        const float top = fmaxf(m, x), base = top == -INFINITY ? 0.0f : top;
        const float f = m == top ? 1.0f : exp2f(m - top), e = exp2f(x - base);
        m = top;
        l = l * f + e;
        o.x = o.x * f + e * v0.x;
        o.y = o.y * f + e * v0.y;
        o.z = o.z * f + e * v1.x;
        o.w = o.w * f + e * v1.y;
    }
}

// Weight of a partial result with maximum m in a whole with maximum top.
__device__ __forceinline__ float join_weight(float m, float top) { return m == -INFINITY ? 0.0f : exp2_approx(m - top); }
#endif  // __CUDACC__

}  // namespace paged
}  // namespace sib
