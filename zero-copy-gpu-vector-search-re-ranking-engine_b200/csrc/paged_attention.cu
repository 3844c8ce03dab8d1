// Host side of zcgvs_paged_attention: argument checks, the choice of kernels and the workspace.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "paged_stream.cuh"

namespace zc {
namespace paged {

namespace {

// Workspace: the status word, then a ticket per CTA, then two partial results per CTA. Sized for
// the largest grid and row tile of any variant.
constexpr int kMaxCtas = 1024;
constexpr size_t kTicketsAt = 256;
constexpr size_t kPartMlAt = kTicketsAt + sizeof(u64) * kMaxCtas;

struct Layout {
    size_t part_o;
    size_t total;
};

// `rows`: of all CTAs' row tiles together.
Layout layout(size_t rows, int padded_dim) {
    Layout l;
    l.part_o = round_up(kPartMlAt + 2 * rows * 2 * sizeof(float), 256);
    l.total = l.part_o + 2 * rows * padded_dim * sizeof(float);
    return l;
}

int padded(int head_dim) { return head_dim <= 64 ? 64 : 128; }

constexpr int kStreamRows = 64;  // largest row tile of the streaming kernel

int stream_ctas(int padded_dim, int sms) { return std::min(kMaxCtas, sms * (padded_dim == 64 ? stream_ctas_per_sm<64>() : stream_ctas_per_sm<128>())); }

std::atomic<uint32_t> g_epoch{0};

uint32_t next_epoch() {
    uint32_t e = ++g_epoch;
    while (e == 0) e = ++g_epoch;  // 0 marks a ticket that was left at zero
    return e;
}

template <typename T, int DP, int WM>
cudaError_t launch_stream(const AttnParams& p, int ctas, cudaStream_t stream) {
    auto kernel = stream_kernel<T, DP, WM>;
    const cudaError_t e = ensure_smem_optin(reinterpret_cast<const void*>(kernel));
    if (e != cudaSuccess) return e;
    KernelTimer timer("paged_stream", stream);
    kernel<<<ctas, kStreamThreads, stream_stages<DP>() * stream_stage_bytes<DP>(), stream>>>(p);
    return cudaGetLastError();
}

template <typename T, int DP>
cudaError_t launch_stream_rows(const AttnParams& p, long long rows, int ctas, cudaStream_t stream) {
    // The smallest row tile that holds a sequence's rows: fewer rows per warp leave warps to split
    // the keys.
    if (rows <= 16) return launch_stream<T, DP, 1>(p, ctas, stream);
    if (rows <= 32) return launch_stream<T, DP, 2>(p, ctas, stream);
    return launch_stream<T, DP, 4>(p, ctas, stream);
}

template <typename T>
cudaError_t launch_stream_any(const AttnParams& p, long long rows, int ctas, cudaStream_t stream) {
    return padded(p.view.head_dim) == 64 ? launch_stream_rows<T, 64>(p, rows, ctas, stream)
                                         : launch_stream_rows<T, 128>(p, rows, ctas, stream);
}

}  // namespace
}  // namespace paged
}  // namespace zc

extern "C" {

size_t zcgvs_paged_attention_workspace_bytes(int head_dim) {
    using namespace zc::paged;
    if (head_dim <= 0 || head_dim > kMaxHeadDim) return 0;
    const int dim = padded(head_dim);
    const size_t sms = static_cast<size_t>(zc::device_sm_count());
    return layout(static_cast<size_t>(stream_ctas(dim, static_cast<int>(sms))) * kStreamRows, dim).total;
}

int zcgvs_paged_attention(const zcgvs_paged_cache* cache, const zcgvs_step_batch* batch, const void* q,
                          int64_t q_token_stride, int64_t q_head_stride, int q_heads, float scale, int causal, int window,
                          void* out, int64_t out_token_stride, int64_t out_head_stride, float* lse, void* workspace,
                          size_t workspace_bytes, void* stream) {
    using namespace zc;
    using namespace zc::paged;
    const char* what = "zcgvs_paged_attention";
    if (cache == nullptr || batch == nullptr) return invalid(what, "null cache or batch");
    if (batch->tokens <= 0 || batch->sequences <= 0 || q_heads <= 0) return ok();
    AttnParams p{};
    int status = make_view(what, cache, batch, p.view);
    if (status != ZCGVS_OK) return status;
    if (q == nullptr || out == nullptr) return invalid(what, "null q or out");
    if (q_heads % cache->kv_heads != 0) return invalid(what, "q_heads must be a multiple of kv_heads");
    status = check_rows(what, "q", q, q_token_stride, q_head_stride);
    if (status == ZCGVS_OK) status = check_rows(what, "out", out, out_token_stride, out_head_stride);
    if (status != ZCGVS_OK) return status;
    if (!std::isfinite(scale)) return invalid(what, "scale must be finite");
    if (window < 0) return invalid(what, "window must be 0 (none) or positive");
    if (batch->max_new < 0) return invalid(what, "max_new must not be negative");
    const int group = q_heads / cache->kv_heads;
    if (static_cast<long long>(batch->tokens) * group > INT_MAX / 2) {
        return invalid(what, "too many tokens and heads for one call");
    }
    const size_t need = zcgvs_paged_attention_workspace_bytes(cache->head_dim);
    if (workspace == nullptr || workspace_bytes < need) {
        return invalid(what, "workspace smaller than zcgvs_paged_attention_workspace_bytes()");
    }
    if (!aligned_to(workspace, 256)) return invalid(what, "workspace must be 256-byte aligned");

    const int dim = padded(cache->head_dim);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.q = static_cast<const uint8_t*>(q);
    p.q_token = q_token_stride;
    p.q_head = q_head_stride;
    p.out = static_cast<uint8_t*>(out);
    p.out_token = out_token_stride;
    p.out_head = out_head_stride;
    p.lse = lse;
    p.q_heads = q_heads;
    p.group = group;
    p.scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
    p.causal = causal != 0;
    p.window = window;
    p.status = reinterpret_cast<uint32_t*>(ws);
    p.tickets = reinterpret_cast<u64*>(ws + kTicketsAt);
    p.part_ml = reinterpret_cast<float*>(ws + kPartMlAt);
    p.epoch = next_epoch();
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const long long rows = static_cast<long long>(std::min(batch->max_new, batch->tokens)) * group;

    const int ctas = stream_ctas(dim, device_sm_count());
    p.part_o = reinterpret_cast<float*>(ws + layout(static_cast<size_t>(ctas) * kStreamRows, dim).part_o);
    p.rows_above = 0;
    p.rows_to = INT_MAX;
    const cudaError_t e = cache->dtype == ZCGVS_DTYPE_F16 ? launch_stream_any<__half>(p, rows, ctas, s)
                                                          : launch_stream_any<__nv_bfloat16>(p, rows, ctas, s);
    if (e != cudaSuccess) return fail_cuda(e, what);
    return ok();
}

}  // extern "C"
