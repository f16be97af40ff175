// paged_abi.cpp -- C ABI of the operators on the paged KV cache
// (include/secure_infer_paged.h): checks of the arguments, tensor maps, launches.
#include "paged.cuh"

#include <climits>
#include <cstring>
#include <mutex>

#define SI_EXPORT extern "C" __attribute__((visibility("default")))

using namespace sib::paged;

namespace {

// The driver's encoder, looked up once; null where there is no driver.
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder()
{
    static std::once_flag once;
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) == cudaSuccess &&
            found == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    });
    return fn;
}

// The encoder wants the device's context, which a host thread only has once it has called the runtime.
template <class... Args>
bool encoded(Args... args)
{
    const auto encode = tensor_map_encoder();
    if (encode == nullptr) return false;
    CUresult e = encode(args...);
    if (int device = 0; e == CUDA_ERROR_INVALID_CONTEXT && cudaGetDevice(&device) == cudaSuccess &&
                        cudaSetDevice(device) == cudaSuccess)
        e = encode(args...);
    return e == CUDA_SUCCESS;
}

bool aligned16(const void* p) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool stride_ok(int64_t elements) { return elements > 0 && elements % 8 == 0 && elements < (int64_t(1) << 38); }

bool pages_ok(const secure_infer_pages* p)
{
    if (p == nullptr || !aligned16(p->k) || !aligned16(p->v) || p->pages == 0 || p->pages > INT_MAX || p->heads == 0 ||
        p->heads > 4096 || p->dtype > SECURE_INFER_FP16)
        return false;
    for (int i = 0; i < 3; ++i)
        if (!stride_ok(p->k_stride[i]) || !stride_ok(p->v_stride[i])) return false;
    return true;
}

bool chunk_ok(const secure_infer_chunk* c)
{
    return c != nullptr && c->block_table != nullptr && c->cu_q != nullptr && c->kv_lens != nullptr && c->seqs > 0 &&
           c->seqs <= (1u << 20) && c->table_width > 0 && c->table_width <= (1u << 23) && c->tokens <= (1u << 28) &&
           c->table_stride >= static_cast<int64_t>(c->table_width);
}

// K or V as [page][head][half of a head][token][64 values]: a box of `tokens`
// tokens lands as [half][token][64], 128-byte rows in the 128-byte swizzle.
bool page_map(CUtensorMap* map, const secure_infer_pages* p, const void* base, const int64_t* stride, uint32_t tokens)
{
    const cuuint64_t dims[5] = {64, kPage, 2, p->heads, p->pages};
    const cuuint64_t bytes[4] = {static_cast<cuuint64_t>(stride[1]) * 2, 128, static_cast<cuuint64_t>(stride[2]) * 2,
                                 static_cast<cuuint64_t>(stride[0]) * 2};
    const cuuint32_t box[5] = {64, tokens, 2, 1, 1}, step[5] = {1, 1, 1, 1, 1};
    const auto type = p->dtype == SECURE_INFER_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return encoded(map, type, 5, const_cast<void*>(base), dims, bytes, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// Queries as [half of a head][token][query head][64 values], in boxes of a KV
// head's group by 128 / group tokens.
bool rows_map(CUtensorMap* map, uint32_t dtype, const void* q, int64_t token_stride, int64_t head_stride, uint32_t tokens,
              uint32_t heads, uint32_t group)
{
    const cuuint64_t dims[4] = {64, heads, tokens, 2};
    const cuuint64_t bytes[3] = {static_cast<cuuint64_t>(head_stride) * 2, static_cast<cuuint64_t>(token_stride) * 2, 128};
    const cuuint32_t box[4] = {64, group, 128 / group, 1}, step[4] = {1, 1, 1, 1};
    const auto type = dtype == SECURE_INFER_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return encoded(map, type, 4, const_cast<void*>(q), dims, bytes, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// Rows per KV head up to which a sequence goes to the kernel for few rows, in
// tiles of eight.  Measured there and in tiles of 128, us: 24 sequences of up to
// 4096 tokens on 8 KV heads with 20 rows 54 and 55, with 24 rows 69 and 57, with
// 32 rows 100 and 53; 8 sequences with 20 rows 27 and 33; 48 of up to 8192 on one
// KV head with 24 rows 34 and 40; one of 300 tokens with 20 rows 7.3 and 14.0.
constexpr uint32_t kFewRows = 24;

// How a call is launched, and the most units of work that its launches may have
// (a page for a tile and a KV head, and what a tile costs besides, in the
// longest context that the table can hold).
struct Work {
    uint32_t group;
    bool tiles;         // sequences of more than kFewRows rows go to the kernel for many
    uint64_t rows_units, tiles_units;

    // Units are counted in 32 bits.
    bool fits() const { return rows_units <= INT_MAX && tiles_units <= INT_MAX; }
};

// What rows see behind a window (0: none) with sinks.
struct Sight {
    int32_t window, sinks;
    Mode mode;
};
Sight sight_of(const secure_infer_chunk& chunk, uint32_t window, uint32_t sinks)
{
    // As many tokens as a table can hold hide nothing, and positions less such a window might pass 32 bits.
    const uint64_t most = static_cast<uint64_t>(chunk.table_width) * kPage;
    if (window == 0 || window >= most || sinks >= most) return {0, 0, kPlain};
    return {static_cast<int32_t>(window), static_cast<int32_t>(sinks), sinks > 0 ? kSinks : kPlain};
}

// Whether sequences that share prefixes fill pairs of tiles.
bool tiles_full(const secure_infer_chunk& chunk, uint64_t group)
{
    return chunk.tokens * group > uint64_t(128) * (chunk.seqs < chunk.tokens ? chunk.seqs : chunk.tokens);
}

// `groups` of sequences share a prefix (kShared): all their rows make tiles of it.
Work work_of(const secure_infer_pages& pages, const secure_infer_chunk& chunk, uint32_t q_heads, Mode mode, uint32_t groups = 0)
{
    Work w{q_heads / pages.heads, false, 0, 0};
    const uint64_t a_tile = rows_cost(mode), a_pair = tiles_cost(mode, tiles_full(chunk, w.group));
    const uint32_t max_q = chunk.max_q == 0 || chunk.max_q > chunk.tokens ? chunk.tokens : chunk.max_q;
    const uint64_t max_rows = static_cast<uint64_t>(max_q) * w.group, rows = static_cast<uint64_t>(chunk.tokens) * w.group;
    // Up to kFewRows rows per KV head a sequence is bound by reading K and V once, which the kernel for few rows does
    // with less latency; more rows are worth tiles of 128.
    w.tiles = (groups > 0 ? rows : max_rows) > kFewRows && w.group <= 128;
    const auto units = [&](uint64_t tiles, uint64_t cost) -> uint64_t {
        return tiles * pages.heads > INT_MAX ? UINT64_MAX : tiles * pages.heads * (chunk.table_width + cost);
    };
    const uint64_t seqs = uint64_t(chunk.seqs) + groups, all = groups > 0 ? 2 * rows : rows;
    if (max_rows > INT_MAX || (groups > 0 && rows > INT_MAX)) w.rows_units = UINT64_MAX;
    else if (!w.tiles) w.rows_units = units(all / 8 + seqs, a_tile);
    else {
        w.rows_units = seqs > 1 ? units(seqs * (kFewRows / 8), a_tile) : 0;
        w.tiles_units = units(all / (2 * (128 / w.group * w.group)) + seqs, a_pair);
    }
    return w;
}

// Whether a call attends what its groups have in common for all their rows at
// once, by what that saves if the common pages are `pages`, all that the table or
// the caller says they may be.  A page takes an SM 4 units of time (1.1 us) for
// eight rows in the kernel for few rows, as long for 128 rows in tiles and 7 for
// 256.  It costs the joining of the parts (0.17 units a row) and, in a call that has
// no tiles otherwise, the tiles' kernel and its own join.  Together and apart, us, in
// a graph: single tokens of 8 KV heads of 4 rows, 2 sequences with 512, 2048 and 8192
// tokens in common 9.7 and 8.3, 12.3 and 9.7, 14.5 and 16.0; 8 sequences with 2048,
// 8192 and 30000 (tiles) 18.3 and 16.1, 23.1 and 31.7, 44.1 and 86.5; 8 chunks of up to
// 40 tokens of 4 rows with 2048, 8192, 30000 33 and 34, 56 and 74, 132 and 249; 5
// chunks of up to 300 tokens of 7 rows with 6144 127 and 108.  Where nothing is said
// of how much is common this stands for the table's width, and is wrong in wide ones:
// 48 single tokens that share nothing 166 and 145.
constexpr int64_t kShareCost = 1000, kShareTilesCost = 12000;
int64_t page_time(uint64_t rows)
{
    return static_cast<int64_t>(rows <= kFewRows ? 4 * ((rows + 7) / 8) : rows <= 128 ? 4 : 7 * ((rows + 255) / 256));
}
// -> the groups that the call's options name, or 0.
uint32_t shared_groups(const secure_infer_pages& pages, const secure_infer_chunk& chunk, uint32_t q_heads,
                       const secure_infer_attend_options* options)
{
    if (options == nullptr || options->plan == nullptr || chunk.tokens == 0 || options->groups == 0) return 0;
    const uint32_t groups = options->groups, most = static_cast<uint32_t>((uint64_t(options->max_common) + kPage - 1) / kPage);
    const uint32_t common = most == 0 || most > chunk.table_width ? chunk.table_width : most;
    const uint64_t group = q_heads / pages.heads, tokens = chunk.tokens, seqs = chunk.seqs < tokens ? chunk.seqs : tokens;
    const int64_t apart = static_cast<int64_t>(seqs) * page_time((tokens + seqs - 1) / seqs * group);
    const int64_t together = groups * page_time((tokens + groups - 1) / groups * group);
    const uint64_t largest = (chunk.max_q == 0 || chunk.max_q > tokens ? tokens : chunk.max_q) * group;
    const int64_t cost = largest > kFewRows || group > 128 || tokens * group <= kFewRows ? kShareCost : kShareTilesCost;
    const double saved = static_cast<double>(apart - together) * common * pages.heads;
    const bool worth = saved > static_cast<double>(cost) + static_cast<double>(tokens * q_heads) / 6;
    return worth && work_of(pages, chunk, q_heads, kShared, groups).fits() ? groups : 0;
}

bool tables_ok(const secure_infer_tables* in, const secure_infer_tables* out)
{
    return in != nullptr && out != nullptr && in->block_table != nullptr && in->lens != nullptr && in->refs != nullptr &&
           out->block_table != nullptr && out->lens != nullptr && out->refs != nullptr && in->seqs > 0 &&
           in->seqs <= (1u << 24) && in->width > 0 && in->width <= (1u << 23) && in->pages > 0 && in->pages <= INT_MAX / 2 &&
           out->seqs == in->seqs && out->width == in->width && out->pages == in->pages &&
           in->block_table != out->block_table && in->lens != out->lens && in->refs != out->refs;
}

bool tensors_ok(const secure_infer_page_tensor* t, uint32_t n, uint64_t page_bytes)
{
    if (t == nullptr || n == 0 || page_bytes == 0 || page_bytes % 16 != 0 || page_bytes > (uint64_t(1) << 30)) return false;
    for (uint32_t i = 0; i < n; ++i)
        if (!aligned16(t[i].base) || t[i].page_stride % 16 != 0 || t[i].page_stride < static_cast<int64_t>(page_bytes))
            return false;
    return true;
}

}  // namespace

SI_EXPORT uint64_t secure_infer_paged_attend_workspace(void) { return attend_workspace_bytes(); }

SI_EXPORT uint64_t secure_infer_capture_id(void* stream)
{
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, &id) != cudaSuccess) {
        cudaGetLastError();   // the legacy stream beside another stream's capture
        return 0;
    }
    return status == cudaStreamCaptureStatusActive ? id : 0;
}

SI_EXPORT int secure_infer_attend_status(void* workspace, uint32_t* status, void* stream)
{
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0 || status == nullptr ||
        secure_infer_capture_id(stream) != 0)
        return -1;
    AttendParams p;
    attend_workspace(workspace, &p);
    const auto st = static_cast<cudaStream_t>(stream);
    uint32_t word = 0;
    if (cudaMemcpyAsync(&word, p.status, sizeof(word), cudaMemcpyDeviceToHost, st) != cudaSuccess ||
        cudaStreamSynchronize(st) != cudaSuccess)
        return -1;
    *status = word != 0;
    return word == 0 || cudaMemsetAsync(workspace, 0, SECURE_INFER_ATTEND_STATE_BYTES, st) == cudaSuccess ? 0 : -1;
}

static bool call_ok(const secure_infer_pages* pages, const secure_infer_chunk* chunk, uint32_t q_heads)
{
    return pages_ok(pages) && chunk_ok(chunk) && q_heads > 0 && q_heads <= (1u << 16) && q_heads % pages->heads == 0;
}

SI_EXPORT int secure_infer_attend_fits(const secure_infer_pages* pages, const secure_infer_chunk* chunk, uint32_t q_heads)
{
    return call_ok(pages, chunk, q_heads) && work_of(*pages, *chunk, q_heads, kPlain).fits();
}

SI_EXPORT int secure_infer_attend_fits_window(const secure_infer_pages* pages, const secure_infer_chunk* chunk,
                                              uint32_t q_heads, uint32_t window, uint32_t sinks)
{
    return call_ok(pages, chunk, q_heads) && work_of(*pages, *chunk, q_heads, sight_of(*chunk, window, sinks).mode).fits();
}

SI_EXPORT uint64_t secure_infer_attend_parts(const secure_infer_pages* pages, const secure_infer_chunk* chunk,
                                             uint32_t q_heads, const secure_infer_attend_options* options)
{
    if (!call_ok(pages, chunk, q_heads) || shared_groups(*pages, *chunk, q_heads, options) == 0) return 0;
    return static_cast<uint64_t>(chunk->tokens) * q_heads * 2 * (kDim + 2) * sizeof(float);
}

// The sequences' common tokens, then the groups, which are read 16 bytes at a time.
static uint64_t group_offset(uint32_t seqs) { return (static_cast<uint64_t>(seqs) + 3) / 4 * 4; }

SI_EXPORT uint64_t secure_infer_shared_prefix_ints(uint32_t seqs, uint32_t groups)
{
    return group_offset(seqs) + static_cast<uint64_t>(groups) * (sizeof(Group) / sizeof(int32_t));
}

SI_EXPORT int secure_infer_shared_prefix(const secure_infer_chunk* chunk, const int32_t* cu_seqs, uint32_t groups,
                                         int32_t* plan, void* stream)
{
    if (!chunk_ok(chunk) || groups == 0 || groups > chunk->seqs || (cu_seqs == nullptr && groups != 1) || !aligned16(plan))
        return -1;
    const PrefixParams p{chunk->block_table, chunk->table_stride, chunk->cu_q, chunk->kv_lens, cu_seqs,
                         static_cast<int32_t>(chunk->table_width), static_cast<int32_t>(chunk->seqs), plan,
                         reinterpret_cast<Group*>(plan + group_offset(chunk->seqs))};
    return launch_shared_prefix(p, groups, static_cast<cudaStream_t>(stream)) == 0 ? 0 : -1;
}

SI_EXPORT int secure_infer_attend_join(const secure_infer_attend_part* parts, uint32_t n, uint32_t tokens, uint32_t heads,
                                       uint32_t dtype, void* out, float* lse, void* stream)
{
    if (parts == nullptr || n == 0 || n > SECURE_INFER_JOIN_PARTS || tokens > (1u << 28) || heads == 0 ||
        heads > (1u << 16) || dtype > SECURE_INFER_FP16)
        return -1;
    if (tokens == 0) return 0;
    if (!aligned16(out) || lse == nullptr || static_cast<uint64_t>(tokens) * heads > (uint64_t(1) << 34)) return -1;
    JoinParams p;
    std::memset(&p, 0, sizeof(p));
    for (uint32_t i = 0; i < n; ++i) {
        const secure_infer_attend_part& a = parts[i];
        if (!aligned16(a.out) || a.lse == nullptr || !stride_ok(a.out_stride[0]) || !stride_ok(a.out_stride[1]) ||
            a.lse_stride[0] < 0 || a.lse_stride[1] < 0)
            return -1;
        p.part[i] = a;
    }
    p.n = static_cast<int32_t>(n);
    p.tokens = static_cast<int32_t>(tokens);
    p.heads = static_cast<int32_t>(heads);
    p.out = out;
    p.lse = lse;
    return launch_join(p, dtype, static_cast<cudaStream_t>(stream)) == 0 ? 0 : -1;
}

SI_EXPORT int secure_infer_paged_attend(const secure_infer_pages* pages, const secure_infer_chunk* chunk, const void* q,
                                        int64_t q_token_stride, int64_t q_head_stride, uint32_t q_heads, void* out,
                                        float* lse, float scale, uint32_t causal, uint32_t window, void* workspace,
                                        void* stream)
{
    return secure_infer_attend(pages, chunk, q, q_token_stride, q_head_stride, q_heads, out, lse, scale, causal, window,
                               nullptr, workspace, stream);
}

SI_EXPORT int secure_infer_attend(const secure_infer_pages* pages, const secure_infer_chunk* chunk, const void* q,
                                  int64_t q_token_stride, int64_t q_head_stride, uint32_t q_heads, void* out, float* lse,
                                  float scale, uint32_t causal, uint32_t window,
                                  const secure_infer_attend_options* options, void* workspace, void* stream)
{
    const uint32_t sinks = options != nullptr ? options->sinks : 0;
    if (!call_ok(pages, chunk, q_heads) || (window != 0 && !causal) || window > INT_MAX || workspace == nullptr ||
        (reinterpret_cast<uintptr_t>(workspace) & 255) != 0 || sinks > INT_MAX || (sinks != 0 && window == 0))
        return -1;
    if (options != nullptr && options->plan != nullptr &&
        (!aligned16(options->plan) || options->groups == 0 || options->groups > chunk->seqs || window != 0))
        return -1;
    if (chunk->tokens == 0) return 0;
    const uint32_t groups = shared_groups(*pages, *chunk, q_heads, options);
    if (!aligned16(q) || !aligned16(out) || !stride_ok(q_token_stride) || !stride_ok(q_head_stride) ||
        (groups > 0 && !aligned16(options->parts)))
        return -1;
    const Sight sight = sight_of(*chunk, window, sinks);
    const Mode mode = groups > 0 ? kShared : sight.mode;
    const Work work = work_of(*pages, *chunk, q_heads, mode, groups);
    if (!work.fits()) return -1;
    const uint32_t group = work.group;

    AttendParams p;
    std::memset(&p, 0, sizeof(p));
    p.q = q;
    p.q_token = q_token_stride;
    p.q_head = q_head_stride;
    p.k = pages->k;
    p.v = pages->v;
    for (int i = 0; i < 3; ++i) {
        p.k_stride[i] = pages->k_stride[i];
        p.v_stride[i] = pages->v_stride[i];
    }
    p.out = out;
    p.lse = lse;
    p.table = chunk->block_table;
    p.table_stride = chunk->table_stride;
    p.cu = chunk->cu_q;
    p.kv = chunk->kv_lens;
    p.width = static_cast<int32_t>(chunk->table_width);
    p.seqs = static_cast<int32_t>(chunk->seqs);
    p.tokens = static_cast<int32_t>(chunk->tokens);
    p.pages = static_cast<int32_t>(pages->pages);
    p.heads = static_cast<int32_t>(pages->heads);
    p.group = static_cast<int32_t>(group);
    p.rows_min = 1;
    p.rows_max = INT_MAX;
    p.causal = causal != 0;
    p.window = sight.window;
    p.sinks = sight.sinks;
    if (groups > 0) {
        p.prefix = options->plan;
        p.shared = reinterpret_cast<const Group*>(options->plan + group_offset(chunk->seqs));
        p.groups = static_cast<int32_t>(groups);
        p.parts = options->parts;
        p.tiles_cost = tiles_cost(kShared, tiles_full(*chunk, group));
    }
    p.scale_log2 = scale * 1.4426950408889634f;
    // Hidden scores are -inf before they are scaled, so the scale is never zero; at 1e-30 all weights are 1.
    if (p.scale_log2 > -1e-30f && p.scale_log2 < 1e-30f) p.scale_log2 = 1e-30f;
    attend_workspace(workspace, &p);
    // At most eight units of work for each of 148 SMs, by the pages that a tile may see.
    const uint64_t rows = static_cast<uint64_t>(chunk->tokens) * group;
    const uint64_t seen = (static_cast<uint64_t>(p.window) + 256 / group) / kPage + 2 + sinks / kPage + 1;
    const uint64_t span = p.window != 0 && seen < chunk->table_width ? seen : chunk->table_width;
    const uint64_t several = rows / (kFewRows + 1) < chunk->seqs ? rows / (kFewRows + 1) : chunk->seqs;
    const uint64_t tiles_most = (groups > 0 ? 2 : 1) * rows / 256 + several + groups + 1;
    p.few_cuts = work.tiles && tiles_most * pages->heads * (span + 2) <= 8 * 148;
    const auto st = static_cast<cudaStream_t>(stream);
    // One call's launches follow one another on the stream: they hand the workspace on.
    static std::mutex launches;
    const std::lock_guard<std::mutex> lock(launches);
    const bool tiles = work.tiles;
    CUtensorMap q_map, k_map, v_map, k_quarters, v_quarters;
    const bool some_rows = !tiles || chunk->seqs > 1;   // (groups go with several sequences)
    if (some_rows && (!page_map(&k_quarters, pages, pages->k, pages->k_stride, 32) ||
                      !page_map(&v_quarters, pages, pages->v, pages->v_stride, 32)))
        return -1;
    if (tiles && (!page_map(&k_map, pages, pages->k, pages->k_stride, kPage) ||
                  !page_map(&v_map, pages, pages->v, pages->v_stride, kPage) ||
                  !rows_map(&q_map, pages->dtype, q, q_token_stride, q_head_stride, chunk->tokens, q_heads, group)))
        return -1;
    AttendParams few = p;
    if (tiles) {
        few.rows_max = kFewRows;
        if (some_rows) p.rows_min = kFewRows + 1;
    }
    if (tiles && some_rows && mode != kPlain) {
        if (launch_attend_both(q_map, k_map, v_map, k_quarters, v_quarters, few, p, mode, pages->dtype, st) != 0) return -1;
    } else {
        few.both = p.both = tiles && some_rows;
        if (some_rows && launch_attend_rows(k_quarters, v_quarters, few, mode, pages->dtype, st) != 0) return -1;
        if (tiles && launch_attend_tiles(q_map, k_map, v_map, p, mode, pages->dtype, st) != 0) return -1;
    }
    return groups > 0 && launch_attend_parts(p, pages->dtype, st) != 0 ? -1 : 0;
}

SI_EXPORT int secure_infer_paged_append(const secure_infer_pages* pages, const secure_infer_chunk* chunk, const void* q,
                                        int64_t q_token_stride, int64_t q_head_stride, uint32_t q_heads, void* q_out,
                                        const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                        int64_t v_token_stride, int64_t v_head_stride, const uint64_t* phase,
                                        const uint32_t* axis, const int32_t* positions, int64_t position_stride,
                                        uint32_t axes, uint32_t interleaved, void* stream)
{
    if (!pages_ok(pages) || !chunk_ok(chunk) || q_heads > (1u << 16) || (phase == nullptr) != (axis == nullptr) ||
        (positions != nullptr && (axes == 0 || axes > 64 || position_stride < 0)))
        return -1;
    if (chunk->tokens == 0) return 0;
    if (!aligned16(k) || !aligned16(v) || !stride_ok(k_token_stride) || !stride_ok(k_head_stride) ||
        !stride_ok(v_token_stride) || !stride_ok(v_head_stride))
        return -1;
    if (q != nullptr && (!aligned16(q) || !aligned16(q_out) || q_heads == 0 || !stride_ok(q_token_stride) ||
                         !stride_ok(q_head_stride)))
        return -1;
    AppendParams p;
    std::memset(&p, 0, sizeof(p));
    p.q = q;
    p.k = k;
    p.v = v;
    p.q_stride[0] = q_token_stride;
    p.q_stride[1] = q_head_stride;
    p.k_in[0] = k_token_stride;
    p.k_in[1] = k_head_stride;
    p.v_in[0] = v_token_stride;
    p.v_in[1] = v_head_stride;
    p.q_out = q_out;
    p.k_cache = pages->k;
    p.v_cache = pages->v;
    for (int i = 0; i < 3; ++i) {
        p.k_stride[i] = pages->k_stride[i];
        p.v_stride[i] = pages->v_stride[i];
    }
    p.table = chunk->block_table;
    p.table_stride = chunk->table_stride;
    p.cu = chunk->cu_q;
    p.kv = chunk->kv_lens;
    p.phase = phase;
    p.axis = axis;
    p.positions = positions;
    p.position_stride = position_stride;
    p.width = static_cast<int32_t>(chunk->table_width);
    p.seqs = static_cast<int32_t>(chunk->seqs);
    p.tokens = static_cast<int32_t>(chunk->tokens);
    p.pages = static_cast<int32_t>(pages->pages);
    p.q_heads = q != nullptr ? static_cast<int32_t>(q_heads) : 0;
    p.heads = static_cast<int32_t>(pages->heads);
    p.axes = axes == 0 ? 1 : static_cast<int32_t>(axes);
    p.interleaved = interleaved != 0;
    return launch_append(p, pages->dtype, static_cast<cudaStream_t>(stream)) == 0 ? 0 : -1;
}

SI_EXPORT uint64_t secure_infer_paged_scratch(const secure_infer_tables* tables, uint32_t n)
{
    return tables == nullptr ? 0 : 4 * table_scratch_ints(tables->seqs, tables->pages, n);
}

SI_EXPORT int secure_infer_paged_copy(const secure_infer_page_tensor* tensors, uint32_t n_tensors, uint64_t page_bytes,
                                      uint32_t pages, const int32_t* src, const int32_t* dst, uint32_t n, void* stream)
{
    if (!tensors_ok(tensors, n_tensors, page_bytes) || pages == 0 || pages > INT_MAX || n > INT_MAX) return -1;
    if (n == 0) return 0;
    if (src == nullptr || dst == nullptr) return -1;
    return launch_page_copy(tensors, n_tensors, page_bytes, pages, src, dst, nullptr, n,
                            static_cast<cudaStream_t>(stream)) == 0
               ? 0
               : -1;
}

SI_EXPORT int secure_infer_paged_fork(const secure_infer_page_tensor* tensors, uint32_t n_tensors, uint64_t page_bytes,
                                      const secure_infer_tables* in, const secure_infer_tables* out,
                                      const int32_t* parents, const int32_t* children, uint32_t n, int32_t* granted,
                                      void* scratch, void* stream)
{
    if (!tensors_ok(tensors, n_tensors, page_bytes) || !tables_ok(in, out) || n > INT_MAX || scratch == nullptr ||
        (n > 0 && (parents == nullptr || children == nullptr || granted == nullptr)))
        return -1;
    const TableParams p{*in, *out, parents, children, granted, nullptr, nullptr, static_cast<int32_t*>(scratch),
                        static_cast<int32_t>(n), 0, 0};
    if (launch_tables(kFork, p, static_cast<cudaStream_t>(stream)) != 0) return -1;
    const CopyList list = table_copy_list(p.scratch, in->pages);
    return launch_page_copy(tensors, n_tensors, page_bytes, in->pages, list.src, list.dst, list.count,
                            n < in->pages ? n : in->pages, static_cast<cudaStream_t>(stream)) == 0
               ? 0
               : -1;
}

SI_EXPORT int secure_infer_paged_reserve(const secure_infer_tables* in, const secure_infer_tables* out,
                                         const int32_t* seqs, const int32_t* new_lens, uint32_t n, int32_t* granted,
                                         void* scratch, void* stream)
{
    if (!tables_ok(in, out) || n > INT_MAX || scratch == nullptr ||
        (n > 0 && (seqs == nullptr || new_lens == nullptr || granted == nullptr)))
        return -1;
    const TableParams p{*in, *out, seqs, new_lens, granted, nullptr, nullptr, static_cast<int32_t*>(scratch),
                        static_cast<int32_t>(n), 0, 0};
    return launch_tables(kReserve, p, static_cast<cudaStream_t>(stream)) == 0 ? 0 : -1;
}

SI_EXPORT int secure_infer_paged_free(const secure_infer_tables* in, const secure_infer_tables* out, const int32_t* seqs,
                                      uint32_t n, void* scratch, void* stream)
{
    if (!tables_ok(in, out) || n > INT_MAX || scratch == nullptr || (n > 0 && seqs == nullptr)) return -1;
    const TableParams p{*in, *out, seqs, nullptr, nullptr, nullptr, nullptr, static_cast<int32_t*>(scratch),
                        static_cast<int32_t>(n), 0, 0};
    return launch_tables(kFree, p, static_cast<cudaStream_t>(stream)) == 0 ? 0 : -1;
}

SI_EXPORT int secure_infer_trim(const secure_infer_tables* in, const secure_infer_tables* out, const int32_t* seqs, uint32_t n,
                                uint32_t window, uint32_t sinks, void* scratch, void* stream)
{
    if (!tables_ok(in, out) || n > INT_MAX || scratch == nullptr || (n > 0 && seqs == nullptr) || window == 0 ||
        window > INT_MAX || sinks > INT_MAX - kPage)
        return -1;
    const TableParams p{*in, *out, seqs, nullptr, nullptr, nullptr, nullptr, static_cast<int32_t*>(scratch),
                        static_cast<int32_t>(n), static_cast<int32_t>(window), static_cast<int32_t>(sinks)};
    return launch_tables(kTrim, p, static_cast<cudaStream_t>(stream)) == 0 ? 0 : -1;
}

SI_EXPORT int secure_infer_paged_compact(const secure_infer_page_tensor* tensors, uint32_t n_tensors,
                                         uint64_t page_bytes, const secure_infer_tables* in,
                                         const secure_infer_tables* out, int32_t* moved, int32_t* live, void* scratch,
                                         void* stream)
{
    if (!tensors_ok(tensors, n_tensors, page_bytes) || !tables_ok(in, out) || moved == nullptr || live == nullptr ||
        scratch == nullptr)
        return -1;
    const TableParams p{*in, *out, nullptr, nullptr, nullptr, moved, live, static_cast<int32_t*>(scratch), 0, 0, 0};
    if (launch_tables(kCompact, p, static_cast<cudaStream_t>(stream)) != 0) return -1;
    const CopyList list = table_copy_list(p.scratch, in->pages);
    return launch_page_copy(tensors, n_tensors, page_bytes, in->pages, list.src, list.dst, list.count, in->pages / 2 + 1,
                            static_cast<cudaStream_t>(stream)) == 0
               ? 0
               : -1;
}
