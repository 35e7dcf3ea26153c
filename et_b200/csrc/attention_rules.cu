// Attention with rules on its scores: the entry point, what it refuses, which kernel a call takes, and the general kernel.
#include <cmath>
#include "attention_rules.h"
#include "common.h"

namespace et {
namespace {

constexpr int kRowWarps = 4;

// A warp to a query of a head: what the tensor-core kernels do not take (heads that are no multiple of 16 or wider than 128, rows that do not start
// on 16 bytes).
__global__ void __launch_bounds__(kRowWarps * 32) attention_rules_rows_kernel(const __grid_constant__ RuleParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x * kRowWarps + (threadIdx.x >> 5), h = blockIdx.y;
    if (row >= p.q_tokens) return;
    int b = row / p.max_q_len;
    if (p.cu_seqlens) {   // the last sequence that starts at or before the row (empty ones start there too)
        int lo = 0, hi = p.batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.cu_seqlens[mid] <= row) lo = mid;
            else hi = mid;
        }
        b = lo;
    }
    if (b >= p.batch) return;
    const RuleSeq s = rule_seq(p, b);
    if (row < s.q0 || row >= s.q0 + s.qlen) return;
    rules_row(p, s, row - s.q0, h);
}

}  // namespace

cudaError_t attention_rules_rows_launch(const RuleParams& p, cudaStream_t st) {
    return launch_pdl(attention_rules_rows_kernel, dim3((p.q_tokens + kRowWarps - 1) / kRowWarps, p.nhead), dim3(kRowWarps * 32), 0, st, p);
}

}  // namespace et

extern "C" size_t et_attention_rules_scratch_size(int batch, int max_k_len) {
    if (batch <= 0 || max_k_len <= 0) return 0;
    return (size_t)batch * (((size_t)max_k_len + 63) / 64) * 8;
}

extern "C" int et_attention_rules(void* out, const void* Q, const void* K, const void* V, int out_pitch, int q_pitch, int k_pitch, int v_pitch,
                                  int nhead, int nhead_kv, int head_dim, const int* cu_seqlens, const int* k_start, const int* k_lens, int batch,
                                  int q_tokens, int k_rows, int max_q_len, int max_k_len, const et_score_rules* rules, void* scratch,
                                  size_t scratch_bytes, void* stream) {
    using namespace et;
    ET_REQUIRE(batch >= 0 && q_tokens >= 0 && k_rows >= 0 && max_q_len >= 0 && max_k_len >= 0, "et_attention_rules: negative size");
    ET_REQUIRE(nhead >= 1 && nhead_kv >= 1 && nhead % nhead_kv == 0, "et_attention_rules: nhead must be a multiple of nhead_kv");
    ET_REQUIRE(head_dim >= 1 && head_dim <= 256, "et_attention_rules: head_dim must be 1 to 256");
    ET_REQUIRE(nhead <= 0xffff && batch <= 0xffffff, "et_attention_rules: too many heads or sequences");
    ET_REQUIRE(max_q_len < kNoLimit && max_k_len < kNoLimit, "et_attention_rules: sequences must be shorter than 2^30");
    ET_REQUIRE(!k_start || k_lens, "et_attention_rules: k_start needs k_lens");
    if (batch == 0 || q_tokens == 0 || max_q_len == 0) return ET_OK;
    ET_REQUIRE(out && Q, "et_attention_rules: null pointer");
    ET_REQUIRE(k_rows == 0 || (K && V), "et_attention_rules: null pointer");
    ET_REQUIRE(cu_seqlens || (long long)batch * max_q_len <= q_tokens, "et_attention_rules: fewer rows than batch x max_q_len");
    ET_REQUIRE(q_pitch >= nhead * head_dim && out_pitch >= nhead * head_dim && k_pitch >= nhead_kv * head_dim && v_pitch >= nhead_kv * head_dim,
               "et_attention_rules: pitch below the width of the heads");
    const et_score_rules none = {0.f, 0.f, nullptr, nullptr, 0, -1, -1, nullptr, nullptr, nullptr};
    const et_score_rules& r = rules ? *rules : none;
    ET_REQUIRE(std::isfinite(r.scale) && r.scale >= 0.f, "et_attention_rules: the scale must be positive");
    ET_REQUIRE(std::isfinite(r.cap) && r.cap >= 0.f, "et_attention_rules: the cap must be positive");
    ET_REQUIRE(!(r.slopes && r.distance_bias), "et_attention_rules: slopes or a table of distances, not both");
    ET_REQUIRE(!r.distance_bias || (r.reach >= 0 && r.reach < kNoLimit), "et_attention_rules: bad reach");
    ET_REQUIRE(!r.q_docs == !r.k_docs, "et_attention_rules: documents of the queries and of the keys, or neither");
    ET_REQUIRE(!r.q_docs || (scratch && scratch_bytes >= et_attention_rules_scratch_size(batch, max_k_len) && (reinterpret_cast<uintptr_t>(scratch) & 7) == 0),
               "et_attention_rules: documents need scratch of et_attention_rules_scratch_size bytes");
    RuleParams p;
    p.out = static_cast<half*>(out); p.q = static_cast<const half*>(Q); p.k = static_cast<const half*>(K); p.v = static_cast<const half*>(V);
    p.out_pitch = out_pitch; p.q_pitch = q_pitch; p.k_pitch = k_pitch; p.v_pitch = v_pitch;
    p.nhead = nhead; p.group = nhead / nhead_kv; p.head_dim = head_dim;
    p.cu_seqlens = cu_seqlens; p.k_start = k_start; p.k_lens = k_lens;
    p.batch = batch; p.q_tokens = q_tokens; p.k_rows = k_rows; p.max_q_len = max_q_len; p.max_k_len = max_k_len;
    const double scale = r.scale > 0.f ? (double)r.scale : 1.0 / std::sqrt((double)head_dim);
    p.scale_log2 = (float)(scale * 1.4426950408889634);
    p.cap_in = r.cap > 0.f ? (float)(2.0 * scale * 1.4426950408889634 / r.cap) : 0.f;
    p.cap_out = (float)(r.cap * 1.4426950408889634);
    p.to_y = r.cap > 0.f ? (float)(scale / r.cap) : 0.f;
    p.cap_near = p.to_y > 0.f ? std::fmin(kCapNear / p.to_y, 3.4e38f) : 0.f;   // (an infinite score is capped)
    p.cap_wide = r.cap > kWideCap;
    ET_REQUIRE(std::isfinite(p.scale_log2) && std::isfinite(p.cap_in) && std::isfinite(p.cap_out), "et_attention_rules: scale and cap are too far apart");
    p.slopes = r.slopes; p.table = static_cast<const half*>(r.distance_bias); p.reach = r.distance_bias ? r.reach : 0;
    p.window_left = r.window_left < 0 || r.window_left >= kNoLimit ? kNoLimit : r.window_left;
    p.window_right = r.window_right < 0 || r.window_right >= kNoLimit ? kNoLimit : r.window_right;
    p.prefix_lens = r.prefix_lens; p.q_docs = r.q_docs; p.k_docs = r.k_docs;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (attention_rules_token_takes(p)) return attention_rules_token_launch(p, st);
    if (attention_rules_tc_takes(p)) return attention_rules_tc_launch(p, p.k_docs ? scratch : nullptr, st);
    return cuda_status(attention_rules_rows_launch(p, st), "et_attention_rules launch");
}

extern "C" int et_attention_rules_by(const et_attention_rules_args* a) {
    ET_REQUIRE(a, "et_attention_rules_by: null pointer");
    return et_attention_rules(a->out, a->Q, a->K, a->V, a->out_pitch, a->q_pitch, a->k_pitch, a->v_pitch, a->nhead, a->nhead_kv, a->head_dim, a->cu_seqlens, a->k_start, a->k_lens,
                              a->batch, a->q_tokens, a->k_rows, a->max_q_len, a->max_k_len, &a->rules, a->scratch, a->scratch_bytes, a->stream);
}
