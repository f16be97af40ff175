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

Work work_of(const secure_infer_pages& pages, const secure_infer_chunk& chunk, uint32_t q_heads)
{
    Work w{q_heads / pages.heads, false, 0, 0};
    const uint32_t max_q = chunk.max_q == 0 || chunk.max_q > chunk.tokens ? chunk.tokens : chunk.max_q;
    const uint64_t max_rows = static_cast<uint64_t>(max_q) * w.group, rows = static_cast<uint64_t>(chunk.tokens) * w.group;
    // Up to kFewRows rows per KV head a sequence is bound by reading K and V once, which the kernel for few rows does
    // with less latency; more rows are worth tiles of 128.
    w.tiles = max_rows > kFewRows && w.group <= 128;
    const auto units = [&](uint64_t tiles, uint64_t cost) -> uint64_t {
        return tiles * pages.heads > INT_MAX ? UINT64_MAX : tiles * pages.heads * (chunk.table_width + cost);
    };
    if (max_rows > INT_MAX) w.rows_units = UINT64_MAX;
    else if (!w.tiles) w.rows_units = units(rows / 8 + chunk.seqs, 1);
    else {
        w.rows_units = chunk.seqs > 1 ? units(uint64_t(chunk.seqs) * (kFewRows / 8), 1) : 0;
        w.tiles_units = units(rows / (2 * (128 / w.group * w.group)) + chunk.seqs, 2);
    }
    return w;
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

SI_EXPORT int secure_infer_attend_fits(const secure_infer_pages* pages, const secure_infer_chunk* chunk, uint32_t q_heads)
{
    return pages_ok(pages) && chunk_ok(chunk) && q_heads > 0 && q_heads <= (1u << 16) && q_heads % pages->heads == 0 &&
           work_of(*pages, *chunk, q_heads).fits();
}

SI_EXPORT int secure_infer_paged_attend(const secure_infer_pages* pages, const secure_infer_chunk* chunk, const void* q,
                                        int64_t q_token_stride, int64_t q_head_stride, uint32_t q_heads, void* out,
                                        float* lse, float scale, uint32_t causal, uint32_t window, void* workspace,
                                        void* stream)
{
    if (!pages_ok(pages) || !chunk_ok(chunk) || q_heads == 0 || q_heads > (1u << 16) ||
        q_heads % pages->heads != 0 || (window != 0 && !causal) || window > INT_MAX || workspace == nullptr ||
        (reinterpret_cast<uintptr_t>(workspace) & 255) != 0)
        return -1;
    if (chunk->tokens == 0) return 0;
    if (!aligned16(q) || !aligned16(out) || !stride_ok(q_token_stride) || !stride_ok(q_head_stride)) return -1;
    const Work work = work_of(*pages, *chunk, q_heads);
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
    // As many tokens as a table can hold hide nothing, and positions less such a window might pass 32 bits.
    p.window = window >= static_cast<uint64_t>(chunk->table_width) * kPage ? 0 : static_cast<int32_t>(window);
    p.scale_log2 = scale * 1.4426950408889634f;
    // Hidden scores are -inf before they are scaled, so the scale is never zero; at 1e-30 all weights are 1.
    if (p.scale_log2 > -1e-30f && p.scale_log2 < 1e-30f) p.scale_log2 = 1e-30f;
    attend_workspace(workspace, &p);
    const auto st = static_cast<cudaStream_t>(stream);
    // One call's launches follow one another on the stream: they hand the workspace on.
    static std::mutex launches;
    const std::lock_guard<std::mutex> lock(launches);
    const bool tiles = work.tiles;
    CUtensorMap q_map, k_map, v_map;
    if (!tiles || chunk->seqs > 1) {
        if (!page_map(&k_map, pages, pages->k, pages->k_stride, 32) || !page_map(&v_map, pages, pages->v, pages->v_stride, 32))
            return -1;
        p.rows_max = tiles ? kFewRows : INT_MAX;
        p.both = tiles;
        if (launch_attend_rows(k_map, v_map, p, pages->dtype, st) != 0) return -1;
        p.rows_min = kFewRows + 1;
        p.rows_max = INT_MAX;
    }
    if (!tiles) return 0;
    if (!page_map(&k_map, pages, pages->k, pages->k_stride, kPage) || !page_map(&v_map, pages, pages->v, pages->v_stride, kPage) ||
        !rows_map(&q_map, pages->dtype, q, q_token_stride, q_head_stride, chunk->tokens, q_heads, group))
        return -1;
    return launch_attend_tiles(q_map, k_map, v_map, p, pages->dtype, st) == 0 ? 0 : -1;
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
                        static_cast<int32_t>(n)};
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
                        static_cast<int32_t>(n)};
    return launch_tables(kReserve, p, static_cast<cudaStream_t>(stream)) == 0 ? 0 : -1;
}

SI_EXPORT int secure_infer_paged_free(const secure_infer_tables* in, const secure_infer_tables* out, const int32_t* seqs,
                                      uint32_t n, void* scratch, void* stream)
{
    if (!tables_ok(in, out) || n > INT_MAX || scratch == nullptr || (n > 0 && seqs == nullptr)) return -1;
    const TableParams p{*in, *out, seqs, nullptr, nullptr, nullptr, nullptr, static_cast<int32_t*>(scratch),
                        static_cast<int32_t>(n)};
    return launch_tables(kFree, p, static_cast<cudaStream_t>(stream)) == 0 ? 0 : -1;
}

SI_EXPORT int secure_infer_paged_compact(const secure_infer_page_tensor* tensors, uint32_t n_tensors,
                                         uint64_t page_bytes, const secure_infer_tables* in,
                                         const secure_infer_tables* out, int32_t* moved, int32_t* live, void* scratch,
                                         void* stream)
{
    if (!tensors_ok(tensors, n_tensors, page_bytes) || !tables_ok(in, out) || moved == nullptr || live == nullptr ||
        scratch == nullptr)
        return -1;
    const TableParams p{*in, *out, nullptr, nullptr, nullptr, moved, live, static_cast<int32_t*>(scratch), 0};
    if (launch_tables(kCompact, p, static_cast<cudaStream_t>(stream)) != 0) return -1;
    const CopyList list = table_copy_list(p.scratch, in->pages);
    return launch_page_copy(tensors, n_tensors, page_bytes, in->pages, list.src, list.dst, list.count, in->pages / 2 + 1,
                            static_cast<cudaStream_t>(stream)) == 0
               ? 0
               : -1;
}
