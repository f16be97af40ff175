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
    int32_t n, kv, q0, part;
};

// What rows see.  The kernels are made for each, so that the usual call does not
// pay for the others.
enum Mode : int {
    kPlain,    // the causal order with or without a window, or every key
    kSinks,    // behind a window the first tokens as well
    kShared    // groups of sequences whose first pages are the same: these are attended once for all of a group's rows
};

// Pages that the beginning and the end of a tile are worth, which the kernels count with its pages and the host when it
// bounds what they count.  Of few rows: with sinks and shared prefixes 2, where 48 answers to 8192 take 45.2 us (1: 50.5,
// 3: 47.6); the usual call keeps the 1 that its results' order of sums goes by.
constexpr int rows_cost(Mode mode) { return mode == kPlain ? 1 : 2; }
// Of a pair of tiles.  With shared prefixes partial results are twice as long, and 4.5 us go besides the pages where
// sequences fill both tiles (`full`).  Eight chunks of up to 40 tokens of 7 rows on 30000: 194 us with 2, 131 with 4; four
// times six drafts of 5 of 8 rows on up to 30000, one tile each: 35.2 and 37.1.
constexpr int kTilesCost = 2, kFullTilesCost = 4;
inline int tiles_cost(Mode mode, bool full) { return mode == kShared && full ? kFullTilesCost : kTilesCost; }

// A group of sequences with a common prefix, as secure_infer_shared_prefix
// leaves it behind the sequences' own prefixes.
struct Group {
    int32_t lead;      // the sequence whose block table is read
    int32_t q0, n;     // the group's new tokens
    int32_t tokens;    // keys in common, whole pages; 0: none
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
    int32_t few_cuts;               // little work for tiles: few of them are cut
    int32_t both;                   // the call has a launch for few rows, and then one for the others, on the same SMs
    int32_t sinks;                  // kSinks: the first tokens that stay visible
    const int32_t* prefix;          // kShared: [seqs] keys in common with the sequence's group
    const Group* shared;            // [groups]
    int32_t groups;
    int32_t tiles_cost;             // tiles_cost() of the call
    float* parts;                   // [2][rows of the output][128] sums over the group's and over a sequence's own keys, then
                                    // [2][rows] maxima and sums of weights
};

// Launchers (cudaError_t values).
int launch_attend_rows(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttendParams& p, Mode mode,
                       uint32_t dtype, cudaStream_t stream);
// q_map: boxes of [128 / group tokens][group heads][64 values].  Not for kShared, which has several sequences.
int launch_attend_tiles(const CUtensorMap& q_map, const CUtensorMap& k_map, const CUtensorMap& v_map,
                        const AttendParams& p, Mode mode, uint32_t dtype, cudaStream_t stream);
// Both kinds of sequences in one launch, not for kPlain.  quarters: the maps of the rows' kernel; few and many: the
// call with the limits of either kind's rows.
int launch_attend_both(const CUtensorMap& q_map, const CUtensorMap& k_map, const CUtensorMap& v_map,
                       const CUtensorMap& k_quarters, const CUtensorMap& v_quarters, const AttendParams& few,
                       const AttendParams& many, Mode mode, uint32_t dtype, cudaStream_t stream);
uint64_t attend_workspace_bytes();
void attend_workspace(void* workspace, AttendParams* p);   // its counters, status word and slots

struct PrefixParams {
    const int32_t* table;
    int64_t table_stride;
    const int32_t* cu;
    const int32_t* kv;
    const int32_t* groups;          // where each begins among the sequences, and the last one's end; null: one of all
    int32_t width, seqs;
    int32_t* prefix;
    Group* shared;
};
int launch_shared_prefix(const PrefixParams& p, uint32_t groups, cudaStream_t stream);
// kShared: makes p.parts into results, after the kernels that leave them.
int launch_attend_parts(const AttendParams& p, uint32_t dtype, cudaStream_t stream);

struct JoinParams {
    secure_infer_attend_part part[SECURE_INFER_JOIN_PARTS];
    int32_t n, tokens, heads;
    void* out;
    float* lse;
};
int launch_join(const JoinParams& p, uint32_t dtype, cudaStream_t stream);

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

enum TableOp : int32_t { kFork, kReserve, kFree, kCompact, kTrim };
struct TableParams {
    secure_infer_tables in, out;
    const int32_t* a;               // fork: parents; reserve, free, trim: sequences
    const int32_t* b;               // fork: children; reserve: new lengths
    int32_t* granted;
    int32_t* moved;
    int32_t* live;
    int32_t* scratch;
    int32_t n;
    int32_t window, sinks;          // trim
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

// The sequence of a token, by a warp: the last s with cu[s] <= token, 32 probes at
// a time.  From L2, since some kernels read them before they have waited.
__device__ __forceinline__ int find_seq(const int32_t* cu, int seqs, int token)
{
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = seqs;   // cu[lo] <= token, and the answer lies in [lo, hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const uint32_t below = __ballot_sync(0xffffffffu, at < hi && __ldcg(cu + at) <= token);
        const int k = below == 0 ? 0 : 31 - __clz(below);
        lo += k * step;
        hi = min(hi, lo + step);
    }
    return lo;
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
//
// Where groups share a prefix, their common keys are sequences of their own
// behind the call's: all new tokens of the group over the prefix, which every
// one of them sees.  What a sequence's rows see besides begins after it.
struct Seq {
    int n, kv, q0;   // new tokens, all tokens, first new token
    // kShared: its first key, which part of its rows this is (0: over a group's keys, 1: over its own, -1: whole), and
    // its row of the block table.
    int begin, part, row;
};

template <int M>
__device__ __forceinline__ int seq_count(const AttendParams& p)
{
    return M == kShared ? p.seqs + p.groups : p.seqs;
}

// A sequence of either launch.
template <int M>
__device__ __forceinline__ Seq load_any(const AttendParams& p, int s)
{
    Seq r;
    r.begin = 0;
    r.part = -1;
    r.row = s;
    if (M == kShared && s >= p.seqs) {
        const int4 g = __ldcg(reinterpret_cast<const int4*>(p.shared) + (s - p.seqs));
        r.row = max(0, min(g.x, p.seqs - 1));
        r.q0 = max(0, min(g.y, p.tokens));
        r.kv = max(0, min(g.w, p.width * kPage));
        r.n = r.kv > 0 ? max(0, min(g.z, p.tokens - r.q0)) : 0;
        r.part = 0;
        return r;
    }
    // From L2, as all that may be read before this kernel has waited for the one before it.
    int a = __ldcg(p.cu + s), b = __ldcg(p.cu + s + 1);
    a = max(0, min(a, p.tokens));
    b = max(a, min(b, p.tokens));
    r.q0 = a;
    r.n = b - a;
    r.kv = max(0, min(__ldcg(p.kv + s), p.width * kPage));
    if (M == kShared) {
        r.begin = max(0, min(__ldcg(p.prefix + s), r.kv));
        r.part = r.begin > 0 ? 1 : -1;
    }
    return r;
}

// Whether this launch takes it.
__device__ __forceinline__ bool is_mine(const AttendParams& p, const Seq& s)
{
    const int64_t rows = static_cast<int64_t>(s.n) * p.group;
    return rows >= p.rows_min && rows <= p.rows_max;
}

template <int M>
__device__ __forceinline__ Seq load_seq(const AttendParams& p, int s)
{
    Seq r = load_any<M>(p, s);
    if (!is_mine(p, r)) r.n = 0;
    return r;
}

struct Span {
    int first, pages;   // page range of a tile
    int lo, hi;         // keys that any row of it sees: [lo, hi), and with sinks min(sinks, hi) before them
    int jump, skip;     // kSinks: from the tile's page `jump` on, `skip` pages behind the sinks are left out

    // Number in its sequence of the tile's page i.
    template <int M>
    __device__ __forceinline__ int page(int i) const
    {
        return first + i + (M == kSinks && i >= jump ? skip : 0);
    }
};

template <int M>
__device__ __forceinline__ bool in_order(const AttendParams& p, const Seq& s)
{
    return p.causal && !(M == kShared && s.part == 0);
}

template <int M>
__device__ __forceinline__ Span tile_span(const AttendParams& p, const Seq& s, int first_token, int last_token)
{
    Span r;
    r.hi = in_order<M>(p, s) ? min(s.kv, s.kv - s.n + last_token + 1) : s.kv;
    if (M == kShared) r.lo = s.begin;
    else r.lo = p.window ? max(0, s.kv - s.n + first_token - p.window + 1) : 0;
    r.jump = r.skip = 0;
    if (r.hi <= r.lo) {
        r.lo = r.hi = r.first = 0;
        r.pages = 1;
    } else {
        r.first = r.lo / kPage;
        r.pages = (r.hi + kPage - 1) / kPage - r.first;
        if (M == kSinks) {
            r.jump = min((min(p.sinks, r.hi) + kPage - 1) / kPage, r.first);
            r.skip = r.first - r.jump;
            r.pages += r.jump;
            r.first = 0;
        }
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

template <int M>
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
        span = tile_span<M>(p, q, first_token, last_token);
    }
    // Its row of the block table.
    __device__ __forceinline__ int row() const { return M == kShared ? q.row : s; }
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
            if (++s >= seq_count<M>(p)) {   // only if lengths changed under the kernel
                left = 0;
                return;
            }
            q = load_seq<M>(p, s);
        } while (q.n == 0);
        tiles = (q.n * p.group + rows_per_tile - 1) / rows_per_tile;
        set_tile(p);
    }
};

// Pages and cost of a tile.
template <int M>
__device__ __forceinline__ int tile_units(const AttendParams& p, const Seq& s, int rows_per_tile, int cost, int tile)
{
    const int r = tile * rows_per_tile;
    return tile_span<M>(p, s, r / p.group, (min(r + rows_per_tile, s.n * p.group) - 1) / p.group).pages + cost;
}

// Up to so many tiles of a sequence are counted by one thread, more by a warp:
// for a chunk of 4096 tokens of 4 rows a count took 4 us by one thread.
constexpr int kOwnTiles = 4;

// Units of every lane's sequence; `largest`: of a tile of theirs.  All lanes call it.
template <int M>
__device__ __forceinline__ int seq_units(const AttendParams& p, const Seq& s, int rows_per_tile, int cost, int& largest)
{
    const int lane = threadIdx.x & 31;
    const int tiles = (s.n * p.group + rows_per_tile - 1) / rows_per_tile;
    int units = 0;
    if (tiles <= kOwnTiles) {
        for (int t = 0; t < tiles; ++t) {
            const int u = tile_units<M>(p, s, rows_per_tile, cost, t);
            units += u;
            largest = max(largest, u);
        }
    }
    for (uint32_t many = __ballot_sync(0xffffffffu, tiles > kOwnTiles); many != 0; many &= many - 1) {
        const int from = __ffs(many) - 1, n = __shfl_sync(0xffffffffu, tiles, from);
        Seq q{__shfl_sync(0xffffffffu, s.n, from), __shfl_sync(0xffffffffu, s.kv, from), 0, 0, -1, 0};
        if (M == kShared) {
            q.begin = __shfl_sync(0xffffffffu, s.begin, from);
            q.part = __shfl_sync(0xffffffffu, s.part, from);
        }
        int sum = 0, most = 0;
        for (int t = lane; t < n; t += 32) {
            const int u = tile_units<M>(p, q, rows_per_tile, cost, t);
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
    int later;    // in one launch: how much later than the other kind's its first scores are there, in the measure of time
};

// SMs for `units` of a kind beside `others` of the other, in launches of their own.
__device__ __forceinline__ int sms_of(const Kind& kind, int units, const Kind& other, int others)
{
    const int grid = gridDim.x;
    if (units == 0 || others == 0 || grid == 1) return grid;
    const float mine = static_cast<float>(units) * kind.time, theirs = static_cast<float>(others) * other.time;
    const int most = max(1, grid * kind.of_16 / 16), least = grid - max(1, grid * other.of_16 / 16);
    return max(max(1, least), min(min(most, grid - 1), __float2int_rn(grid * (mine / (mine + theirs)))));
}

// SMs for units of few rows beside units of many in one launch: both end together
// where few / x = many / (grid - x) + later, a quadratic equation.
__device__ __forceinline__ int sms_for_few(const Kind& few, int units, const Kind& many, int others)
{
    const int grid = gridDim.x;
    if (units == 0 || others == 0 || grid == 1) return units == 0 ? 0 : grid;
    const float u = static_cast<float>(units) * few.time, v = static_cast<float>(others) * many.time;
    const float later = many.later, b = u + v + later * grid;
    const float x = 2.0f * u * grid / (b + sqrtf(fmaxf(0.0f, b * b - 4.0f * later * u * grid)));
    // The whole number on either side with the earlier end.
    const int most = max(1, min(grid * few.of_16 / 16, grid - 1)), low = max(1, min(most, __float2int_rd(x)));
    const int high = min(most, low + 1);
    const auto end = [&](int r) { return fmaxf(u / r, v / (grid - r) + later); };
    return end(high) < end(low) ? high : low;
}

// All threads of the block take part; `warp_sums` holds three values per warp.
// Where no tile has more than `whole` units a CTA gets the largest one's:
// cutting it would cost more than the few pages that it would save.  Where the
// call has work of both kinds each gets SMs by the time that its units take:
// the first CTAs of a launch work and the others leave theirs to the other
// launch, so reading pages for few rows goes on beside the products of many: 333
// tokens after 2167 and 15 single tokens of up to 4000 take 53 us, 62 one kind
// after the other.
template <int kThreads, int M>
__device__ __forceinline__ void find_share(const AttendParams& p, const Kind& kind, const Kind& other, Share* share,
                                           int32_t* warp_sums)
{
    const int rows_per_tile = kind.rows_per_tile, cost = kind.cost, whole = kind.whole;
    constexpr int kWarps = kThreads / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, seqs = seq_count<M>(p);
    const int down = tid == 0 ? static_cast<int>(__ldcg(p.status)) : 0;
    Share r;
    r.begin = r.total = 0;
    // The first pass sums the units, the second finds the sequence that holds this CTA's first; where every sequence
    // has a thread one pass does both.
    const bool one = seqs <= kThreads;
    for (int pass = one ? 1 : 0; pass < 2; ++pass) {
        int base = 0, largest = 0, others = 0;
        for (int s0 = 0; s0 < seqs; s0 += kThreads) {
            const int s = s0 + tid;
            Seq q{};
            int own_largest = 0, unused = 0, beside = 0;
            if (s < seqs) q = load_any<M>(p, s);
            Seq o = q;
            if (is_mine(p, q)) o.n = 0;
            else q.n = 0;
            if (p.both && (one || pass == 0)) {
                beside = __reduce_add_sync(0xffffffffu, seq_units<M>(p, o, other.rows_per_tile, other.cost, unused));
            }
            const int own = seq_units<M>(p, q, rows_per_tile, cost, own_largest);
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
            // A lane per warp.
            static_assert(kWarps <= 32, "a warp sums the warps");
            const bool has = lane < kWarps;
            const int x = has ? warp_sums[lane] : 0;
            const int before = base + __reduce_add_sync(0xffffffffu, lane < warp ? x : 0);
            base += __reduce_add_sync(0xffffffffu, x);
            largest = max(largest, __reduce_max_sync(0xffffffffu, has ? warp_sums[kWarps + lane] : 0));
            others += __reduce_add_sync(0xffffffffu, has ? warp_sums[2 * kWarps + lane] : 0);
            if (one || (pass == 0 && s0 + kThreads >= seqs)) {
                r.total = base;
                r.ctas = max(1, min(sms_of(kind, base, other, others), largest <= whole ? base / max(1, largest) : base));
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

// The same for one launch of both kinds: its first CTAs take the tiles of few rows,
// its last ones those of many, counted from the end.  -> whether this one takes
// the former.  few and many: the call as either kind sees it.
template <int kThreads, int M>
__device__ __forceinline__ bool find_share_of_both(const AttendParams& few, const Kind& few_kind, const AttendParams& many,
                                                   const Kind& many_kind, Share* share, int32_t* warp_sums, int& cta)
{
    constexpr int kWarps = kThreads / 32;
    static_assert(kWarps <= 32, "a warp sums the warps");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, seqs = seq_count<M>(few);
    const int down = tid == 0 ? static_cast<int>(__ldcg(few.status)) : 0;
    Share r;
    r.begin = r.total = r.units = 0;
    bool first_kind = true;
    cta = blockIdx.x;
    const bool one = seqs <= kThreads;
    for (int pass = one ? 1 : 0; pass < 2; ++pass) {
        int base = 0, all_few = 0, all_many = 0, largest = 0;
        for (int s0 = 0; s0 < seqs; s0 += kThreads) {
            const int s = s0 + tid;
            Seq q{};
            int own_largest = 0, unused = 0;
            if (s < seqs) q = load_any<M>(few, s);
            Seq f = q, m = q;
            if (!is_mine(few, q)) f.n = 0;
            if (!is_mine(many, q)) m.n = 0;
            const int few_units = seq_units<M>(few, f, few_kind.rows_per_tile, few_kind.cost, own_largest);
            const int many_units = seq_units<M>(many, m, many_kind.rows_per_tile, many_kind.cost, unused);
            const int few_sum = __reduce_add_sync(0xffffffffu, few_units), many_sum = __reduce_add_sync(0xffffffffu, many_units);
            own_largest = __reduce_max_sync(0xffffffffu, own_largest);
            if (lane == 0) {
                warp_sums[warp] = few_sum;
                warp_sums[kWarps + warp] = own_largest;
                warp_sums[2 * kWarps + warp] = many_sum;
            }
            __syncthreads();
            const bool has = lane < kWarps;
            const int x = has ? warp_sums[lane] : 0, y = has ? warp_sums[2 * kWarps + lane] : 0;
            all_few += __reduce_add_sync(0xffffffffu, x);
            all_many += __reduce_add_sync(0xffffffffu, y);
            largest = max(largest, __reduce_max_sync(0xffffffffu, has ? warp_sums[kWarps + lane] : 0));
            if (one || (pass == 0 && s0 + kThreads >= seqs)) {
                const int sms = sms_for_few(few_kind, all_few, many_kind, all_many), grid = gridDim.x;
                const int few_ctas = min(sms, largest <= few_kind.whole ? all_few / max(1, largest) : all_few);
                first_kind = static_cast<int>(blockIdx.x) < few_ctas;
                cta = first_kind ? blockIdx.x : grid - 1 - blockIdx.x;
                r.total = first_kind ? all_few : all_many;
                r.ctas = first_kind ? few_ctas : max(1, min(grid - sms, all_many));
                r.per = r.total / r.ctas;
                r.more = r.total - r.per * r.ctas;
                r.begin = r.begin_of(cta);
                r.units = cta < r.ctas ? r.per + (cta < r.more) : 0;
                if (tid == 0) {
                    r.seq = -1;
                    r.seq_unit = 0;
                    r.down = down;
                    *share = r;
                }
                __syncthreads();
            }
            if (pass == 1) {
                const int own = first_kind ? few_units : many_units, z = first_kind ? x : y;
                int sum = own;
                for (int d = 1; d < 32; d <<= 1) {
                    const int up = __shfl_up_sync(0xffffffffu, sum, d);
                    if (lane >= d) sum += up;
                }
                const int first = base + __reduce_add_sync(0xffffffffu, lane < warp ? z : 0) + sum - own;
                if (r.units > 0 && own > 0 && r.begin >= first && r.begin < first + own) {
                    share->seq = s;
                    share->seq_unit = first;
                    share->q = q;
                }
                base += __reduce_add_sync(0xffffffffu, z);
            }
            __syncthreads();
        }
    }
    return first_kind;
}

// All lanes of a warp call it.
template <int M>
__device__ __forceinline__ Walk<M> start_walk(const AttendParams& p, int rows_per_tile, int cost, const Share& share)
{
    Walk<M> w;
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
        int upto = t < w.tiles ? tile_units<M>(p, w.q, rows_per_tile, cost, t) * p.heads : 0;
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

// Keys that row r of the tile sees: [lo, hi], and with sinks those before
// min(sinks, hi + 1).
template <int M>
__device__ __forceinline__ void row_keys(const AttendParams& p, const Seq& s, int token, int& lo, int& hi)
{
    hi = in_order<M>(p, s) ? min(s.kv, s.kv - s.n + token + 1) - 1 : s.kv - 1;
    if (M == kShared) lo = s.begin;
    else lo = p.window ? max(0, s.kv - s.n + token - p.window + 1) : 0;
}

// Keys that a row sees on `pages` of its tile's pages from page `from` on: [a, b),
// and with sinks [sa, sb) before them.
struct PieceKeys {
    int sa, sb, a, b;
};
template <int M>
__device__ __forceinline__ PieceKeys piece_keys(const AttendParams& p, const Span& span, int from, int pages, int lo, int hi)
{
    PieceKeys k{0, 0, 0, 0};
    if (M != kSinks) {
        const int first = span.page<M>(from) * kPage;
        k.a = max(lo, first);
        k.b = min(hi + 1, first + pages * kPage);
        return k;
    }
    // With pages left out the piece is what lies before them and what lies behind.
    const int end = from + pages;
    k.sa = from * kPage;
    k.sb = min(min(min(p.sinks, lo), hi + 1), (span.skip > 0 ? min(end, span.jump) : end) * kPage);
    k.a = max(lo, (span.skip > 0 ? max(from, span.jump) + span.skip : from) * kPage);
    k.b = min(hi + 1, (end + span.skip) * kPage);
    return k;
}

// One row over the keys `in` by one warp, straight from the pages: lane l holds
// values 4l .. 4l+3.  Only rows of a tile in which some row must not see an
// infinite or NaN value that another one does see come here: in a matrix
// product zero times such a value would be NaN.  A key takes about 430
// clocks, the rows of a long piece longer than the other warps' waits last, so
// it counts its way in *work.
template <typename T, int M>
__device__ __forceinline__ void row_by_definition_here(const AttendParams& p, const T* q, const int32_t* table, int head,
                                                       PieceKeys in, float& m, float& l, float4& o, volatile int* work)
{
    const int d = 4 * (threadIdx.x & 31);
    const uint2 qx = __ldcg(reinterpret_cast<const uint2*>(q + d));
    const float2 q0 = unpack2<T>(qx.x), q1 = unpack2<T>(qx.y);
    m = -INFINITY;
    l = 0.0f;
    o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int sinks = M == kSinks ? max(0, in.sb - in.sa) : 0, keys = sinks + max(0, in.b - in.a);
    for (int i = 0; i < keys; ++i) {
        if ((i & 1023) == 0 && d == 0) atomicAdd(const_cast<int*>(work), 1);
        const int j = i < sinks ? in.sa + i : in.a + i - sinks;
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

template <typename T, int M>
__device__ __noinline__ void row_by_definition(const AttendParams& p, const T* q, const int32_t* table, int head,
                                               PieceKeys in, float& m, float& l, float4& o, volatile int* work)
{
    row_by_definition_here<T, M>(p, q, table, head, in, m, l, o, work);
}

// One row's result, by a warp: values 4 lane .. 4 lane + 3 of the sum x, the
// maximum and the sum of weights; `none`: it sees no key.  Where a group's common
// keys are attended elsewhere it goes to the parts, as it is.
template <typename T, int M>
__device__ __forceinline__ void put_row(const AttendParams& p, int part, int64_t at, float4 x, float top, float sum, bool none)
{
    const int lane = threadIdx.x & 31;
    if (M == kShared && part >= 0) {
        const int64_t rows = static_cast<int64_t>(p.tokens) * p.heads * p.group, to = part * rows + at;
        *reinterpret_cast<float4*>(p.parts + to * kDim + lane * 4) = x;
        if (lane == 0) *reinterpret_cast<float2*>(p.parts + 2 * rows * kDim + 2 * to) = make_float2(top, sum);
        return;
    }
    const float inv = 1.0f / sum;
    uint2 packed = make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
    if (none) packed = make_uint2(0, 0);
    *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at * kDim + lane * 4) = packed;
    if (p.lse != nullptr && lane == 0) p.lse[at] = none ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// Weight of a partial result with maximum m in a whole with maximum top.
__device__ __forceinline__ float join_weight(float m, float top) { return m == -INFINITY ? 0.0f : exp2_approx(m - top); }
#endif  // __CUDACC__

}  // namespace paged
}  // namespace sib
