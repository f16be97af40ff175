// paged_join.cu -- attention over parts of the keys made into attention over
// all of them, and the finding of the prefixes that sequences share:
//
//   lse = log sum_i e^lse_i,  out = sum_i e^(lse_i - lse) out_i.
#include "paged.cuh"
#include "gcm_kernels.cuh"

namespace sib {
namespace paged {
namespace {

// ------------------------------------------------------------ shared prefixes
//
// A block per group.  A page is common when every sequence of the group that has
// new tokens names it in the same place, and all of its tokens lie before the
// first new one of each: every new token sees all of them.  A thread compares a
// column of the sequences' rows with the first one's, 64 columns at a time until
// one differs, eight rows on their way at once.  Once a step for all its layers:
// bound by the latency of its reads.  Measured: 48 sequences with 64 pages in common
// 3.4 us, four groups of six with up to 234 4.5, 1024 with 64 17 (78 by a warp a row).
constexpr int kPrefixThreads = 1024;
constexpr int kPrefixColumns = 64;

__global__ void __launch_bounds__(kPrefixThreads) shared_prefix_kernel(const __grid_constant__ PrefixParams p)
{
    __shared__ int first, end, lead, members, common;
    const int tid = threadIdx.x, g = blockIdx.x;
    wait_for_earlier_kernels();
    dependents_may_launch();
    if (tid == 0) {
        first = end = 0;
        lead = INT32_MAX;
        members = 0;
        common = p.width;
    }
    __syncthreads();
    // Groups follow one another whatever the list holds, so a sequence is in one at most.
    auto bound = [&](int i) {
        const int all = p.groups == nullptr ? (i == 0 ? 0 : p.seqs) : p.groups[i];
        return max(0, min(all, p.seqs));
    };
    for (int i = tid; i <= g + 1; i += kPrefixThreads) {
        const int at = bound(i);
        if (i <= g) atomicMax(&first, at);
        atomicMax(&end, at);
    }
    __syncthreads();
    auto new_tokens = [&](int s) {
        const int q0 = max(0, p.cu[s]);
        return max(q0, p.cu[s + 1]) - q0;
    };
    for (int s = first + tid; s < end; s += kPrefixThreads) {
        const int n = new_tokens(s);
        if (n == 0) continue;
        atomicMin(&lead, s);
        atomicAdd(&members, 1);
        atomicMin(&common, max(0, min(p.kv[s], p.width * kPage) - n) / kPage);
    }
    __syncthreads();
    if (members > 1) {
        constexpr int kRowsAtOnce = kPrefixThreads / kPrefixColumns;
        for (int c0 = 0; c0 < common; c0 += kPrefixColumns) {
            const int c = c0 + tid % kPrefixColumns;
            bool differs = false;
            if (c < common) {
                const int32_t page = p.table[lead * p.table_stride + c];
#pragma unroll 8
                for (int s = first + tid / kPrefixColumns; s < end; s += kRowsAtOnce)
                    differs |= p.table[s * p.table_stride + c] != page && new_tokens(s) != 0;
            }
            __syncthreads();   // all have read how many there are
            if (differs) atomicMin(&common, c);
            __syncthreads();
        }
    }
    __syncthreads();
    const int tokens = members > 1 ? common * kPage : 0;
    for (int s = first + tid; s < end; s += kPrefixThreads) p.prefix[s] = tokens;
    // Sequences of no group.
    if (g == 0)
        for (int s = tid; s < first; s += kPrefixThreads) p.prefix[s] = 0;
    if (g == static_cast<int>(gridDim.x) - 1)
        for (int s = end + tid; s < p.seqs; s += kPrefixThreads) p.prefix[s] = 0;
    if (tid == 0) {
        const int q0 = tokens > 0 ? max(0, p.cu[first]) : 0;
        p.shared[g] = Group{tokens > 0 ? lead : 0, q0, tokens > 0 ? max(q0, p.cu[end]) - q0 : 0, tokens};
    }
}

// ------------------------------------------------- a group's keys and a row's own
//
// (m, l, o) over the group's pages and over the sequence's own keys join by the rule
// that joins pieces.  A warp per row of the output, which finds its sequence while
// the kernels before go on; rows of sequences that share nothing are whole already.
// Bound by latency: 2 to 3 us behind the kernels for 48 tokens of 32 heads.
constexpr int kPartsWarps = 8;

template <typename T>
__global__ void __launch_bounds__(32 * kPartsWarps) attend_parts_kernel(const __grid_constant__ AttendParams p)
{
    const int lane = threadIdx.x & 31, token = blockIdx.x, head = blockIdx.y * kPartsWarps + (threadIdx.x >> 5);
    const int heads = p.heads * p.group;
    // What the call was given was complete before its first kernel read it.
    const Seq q = load_seq<kShared>(p, find_seq(p.cu, p.seqs, token));
    wait_for_earlier_kernels();
    dependents_may_launch();
    if (head >= heads || q.part != 1 || token < q.q0 || token >= q.q0 + q.n) return;
    const int64_t rows = static_cast<int64_t>(p.tokens) * heads, at = static_cast<int64_t>(token) * heads + head;
    float4 x[2];
    float2 stat[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        x[i] = __ldcg(reinterpret_cast<const float4*>(p.parts + (i * rows + at) * kDim) + lane);
        stat[i] = __ldcg(reinterpret_cast<const float2*>(p.parts + 2 * rows * kDim) + i * rows + at);
    }
    const float top = fmaxf(stat[0].x, stat[1].x), f0 = join_weight(stat[0].x, top), f1 = join_weight(stat[1].x, top);
    const float4 sum = make_float4(f0 * x[0].x + f1 * x[1].x, f0 * x[0].y + f1 * x[1].y, f0 * x[0].z + f1 * x[1].z,
                                   f0 * x[0].w + f1 * x[1].w);
    put_row<T, kPlain>(p, -1, at, sum, top, f0 * stat[0].y + f1 * stat[1].y, false);
}

// ---------------------------------------------------------------------- parts
//
// Bound by reading every part's rows and writing one's.  Sixteen lanes a row,
// 16-byte accesses, every part on its way at once.  Measured: three parts of 8000
// tokens of 28 heads 37.7 us in a graph, where a part of the inputs is in L2, and 41.4
// by calls with cold ones, 5.6 TB/s, where the copy rate would take 35.7; two of 16
// tokens 1.6 and 6.0, which is the host's time.
constexpr int kJoinPartsThreads = 256;
constexpr int kJoinPartsRows = kJoinPartsThreads / 16;

template <typename T, int kParts>
__global__ void __launch_bounds__(kJoinPartsThreads) join_parts_kernel(const __grid_constant__ JoinParams p)
{
    const int sub = threadIdx.x & 15;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kJoinPartsRows + (threadIdx.x >> 4);
    wait_for_earlier_kernels();
    dependents_may_launch();
    if (row >= static_cast<int64_t>(p.tokens) * p.heads) return;
    const int64_t token = row <= UINT32_MAX ? static_cast<uint32_t>(row) / static_cast<uint32_t>(p.heads) : row / p.heads;
    const int64_t head = row - token * p.heads;
    uint4 x[kParts];
    float lse[kParts];
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
        const secure_infer_attend_part& part = p.part[i];
        lse[i] = part.lse[token * part.lse_stride[0] + head * part.lse_stride[1]];
        x[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(part.out) + token * part.out_stride[0] +
                                               head * part.out_stride[1] + sub * 8);
    }
    float top = lse[0];   // NaN where one of them is, which fmaxf would pass over: the row failed then
#pragma unroll
    for (int i = 1; i < kParts; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(lse[i]));
    const float base = top == -INFINITY ? 0.0f : top;
    float total = 0.0f, y[8] = {};
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
        if (lse[i] == -INFINITY) continue;   // a part of which the row sees nothing counts for nothing, whatever it holds
        const float w = exp2f((lse[i] - base) * 1.4426950408889634f);
        total += w;
        const uint32_t v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 u = unpack2<T>(v[j]);
            y[2 * j] += w * u.x;
            y[2 * j + 1] += w * u.y;
        }
    }
    const float inv = top == -INFINITY ? 0.0f : 1.0f / total;
    // Rounded once, to the type of the parts.
    *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row * kDim + sub * 8) =
        make_uint4(pack2<T>(y[0] * inv, y[1] * inv), pack2<T>(y[2] * inv, y[3] * inv), pack2<T>(y[4] * inv, y[5] * inv),
                   pack2<T>(y[6] * inv, y[7] * inv));
    if (sub == 0) p.lse[row] = top == -INFINITY ? -INFINITY : base + logf(total);
}

template <class... Args>
cudaError_t launch(void (*kernel)(Args...), dim3 grid, int threads, KernelKind kind, cudaStream_t stream, const Args&... args)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    ProfileScope prof(kind, stream);
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace

int launch_shared_prefix(const PrefixParams& p, uint32_t groups, cudaStream_t stream)
{
    return launch(shared_prefix_kernel, dim3(groups), kPrefixThreads, kKernSharedPrefix, stream, p);
}

int launch_attend_parts(const AttendParams& p, uint32_t dtype, cudaStream_t stream)
{
    AttendParams all = p;
    all.rows_min = 1;   // sequences of both kinds
    all.rows_max = INT32_MAX;
    const dim3 grid(p.tokens, (p.heads * p.group + kPartsWarps - 1) / kPartsWarps);
    const auto kernel = dtype == SECURE_INFER_FP16 ? attend_parts_kernel<__half> : attend_parts_kernel<__nv_bfloat16>;
    return launch(kernel, grid, 32 * kPartsWarps, kKernAttendParts, stream, all);
}

template <typename T>
static int launch_join_parts(const JoinParams& p, cudaStream_t stream)
{
    const int64_t blocks = (static_cast<int64_t>(p.tokens) * p.heads + kJoinPartsRows - 1) / kJoinPartsRows;
    if (blocks > INT32_MAX) return cudaErrorInvalidValue;
    // A kernel for each number of parts: three in one made for up to four took 41.4 us where three alone take 37.5.
    using Kernel = void (*)(const JoinParams);
    static constexpr Kernel kernels[SECURE_INFER_JOIN_PARTS] = {
        join_parts_kernel<T, 1>, join_parts_kernel<T, 2>, join_parts_kernel<T, 3>, join_parts_kernel<T, 4>,
        join_parts_kernel<T, 5>, join_parts_kernel<T, 6>, join_parts_kernel<T, 7>, join_parts_kernel<T, 8>};
    const Kernel kernel = kernels[p.n - 1];
    return launch(kernel, dim3(static_cast<uint32_t>(blocks)), kJoinPartsThreads, kKernJoinParts, stream, p);
}

int launch_join(const JoinParams& p, uint32_t dtype, cudaStream_t stream)
{
    return dtype == SECURE_INFER_FP16 ? launch_join_parts<__half>(p, stream) : launch_join_parts<__nv_bfloat16>(p, stream);
}

}  // namespace paged
}  // namespace sib
