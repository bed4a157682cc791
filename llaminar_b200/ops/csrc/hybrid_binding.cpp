// Python bindings of the hybrid family's blocks: an extension of its own, so that a process that serves another family neither compiles
// nor loads it.  Every argument is checked on the host before a launch.
#include <c10/cuda/CUDAGuard.h>

#include <cfloat>

#include "binding_util.h"
#include "hybrid.h"
#include "launch.h"

namespace {
using namespace llm_binding;

void same_device(const Tensor& a, const Tensor& b, const char* name) { TORCH_CHECK(b.is_cuda() && b.device() == a.device(), name, " must be on the device of the rows"); }

// Rows whose values lie next to one another, in bf16
const __nv_bfloat16* bf16_rows(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == torch::kBFloat16 && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)), name, " must be bf16 rows on the GPU");
    return reinterpret_cast<const __nv_bfloat16*>(t.data_ptr());
}
const float* floats_on(const Tensor& like, const Tensor& t, int64_t n, const char* name) {
    same_device(like, t, name);
    return floats(t, n, name);
}
const int* ints_on(const Tensor& like, const Tensor& t, int64_t n, const char* name) {
    same_device(like, t, name);
    TORCH_CHECK(t.numel() == n, name, " must hold ", std::to_string(n), " values");
    return ints(t, name);
}

// The state pools and sizes; C counts the channels of q | k | v
llm::GdnParams gdn_state(const Tensor& conv, const Tensor& rec, int64_t n_k) {
    llm::GdnParams p = {};
    want(conv, torch::kFloat32, "conv_state"); want(rec, torch::kFloat32, "rec");
    TORCH_CHECK(conv.dim() == 3 && rec.dim() == 4 && rec.size(2) == rec.size(3) && conv.size(0) == rec.size(0), "conv_state must be [slots, C, K - 1] and rec [slots, n_v, d, d]");
    same_device(rec, conv, "conv_state");
    p.n_slots = rec.size(0); p.n_v = rec.size(1); p.d = rec.size(2); p.n_k = n_k; p.C = conv.size(1); p.K = conv.size(2) + 1;
    TORCH_CHECK(p.d == 32 || p.d == 64 || p.d == 128, "head size must be 32, 64 or 128");
    TORCH_CHECK(p.n_k >= 1 && p.n_v >= 1 && p.n_v <= 65535 && p.C == (2 * p.n_k + p.n_v) * p.d, "conv_state must have (2 n_k + n_v) d channels");
    TORCH_CHECK(p.K >= 2 && p.K <= 16, "the convolution must have 2 to 16 taps");
    TORCH_CHECK(reinterpret_cast<uintptr_t>(rec.data_ptr()) % 16 == 0, "rec must be 16-byte aligned");
    p.conv = conv.data_ptr<float>(); p.rec = rec.data_ptr<float>();
    return p;
}

llm::GdnParams gdn_params(const Tensor& in, int64_t C, int64_t z_off, int64_t ab_off, const Tensor& conv_w, const Tensor& ssm_a, const Tensor& dt_bias, const Tensor& norm_w,
                          const Tensor& conv, const Tensor& rec, const Tensor& slots, const Tensor& out, int64_t n_k, int64_t v_head_offset, double eps) {
    llm::GdnParams p = gdn_state(conv, rec, n_k);
    p.in = bf16_rows(in, "in");
    same_device(in, rec, "rec"); same_device(in, out, "out");
    TORCH_CHECK(C == p.C && z_off >= 0 && ab_off >= 0 && z_off + (int64_t)p.n_v * p.d <= in.size(1) && ab_off + 2 * (int64_t)p.n_v <= in.size(1) && C <= in.size(1),
                "in: columns of q | k | v, z or alpha | beta are missing");
    TORCH_CHECK(in.size(0) <= INT32_MAX && in.stride(0) <= INT32_MAX, "in: too many rows");
    p.in_row = in.stride(0); p.n_rows = in.size(0); p.z_off = z_off; p.ab_off = ab_off;
    TORCH_CHECK(conv_w.dim() == 2 && conv_w.size(1) == p.K, "conv_w must be [C, K]");
    p.conv_w = floats_on(in, conv_w, (int64_t)p.C * p.K, "conv_w");
    p.ssm_a = floats_on(in, ssm_a, p.n_v, "ssm_a"); p.dt_bias = floats_on(in, dt_bias, p.n_v, "dt_bias"); p.norm_w = floats_on(in, norm_w, p.d, "norm_w");
    p.n_seqs = slots.numel();
    TORCH_CHECK(p.n_seqs <= 65535, "more than 65535 sequences");
    p.slots = ints_on(in, slots, p.n_seqs, "slots");
    bf16_rows(out, "out");
    TORCH_CHECK(out.size(0) == in.size(0) && out.size(1) == (int64_t)p.n_v * p.d, "out must be [rows, n_v d]");
    p.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr()); p.out_row = out.stride(0);
    TORCH_CHECK(v_head_offset >= 0 && v_head_offset <= INT32_MAX / 2, "v_head_offset");
    p.v_head_offset = v_head_offset; p.eps = eps;
    return p;
}

int gdn_prefill(const Tensor& in, int64_t C, int64_t z_off, int64_t ab_off, const Tensor& conv_w, const Tensor& ssm_a, const Tensor& dt_bias, const Tensor& norm_w,
                const Tensor& conv, const Tensor& rec, const Tensor& positions, const Tensor& cu, const Tensor& slots, const Tensor& out, int64_t n_k, int64_t v_head_offset, double eps,
                const OptTensor& workspace, const OptTensor& status) {
    llm::GdnParams p = gdn_params(in, C, z_off, ab_off, conv_w, ssm_a, dt_bias, norm_w, conv, rec, slots, out, n_k, v_head_offset, eps);
    p.positions = ints_on(in, positions, in.size(0), "positions");
    p.cu = ints_on(in, cu, p.n_seqs + 1, "cu");
    const c10::cuda::CUDAGuard guard(in.device());
    int launches = 1;
    if (workspace) {
        same_device(in, *workspace, "workspace");
        want(*workspace, torch::kUInt8, "workspace");
        TORCH_CHECK(status.has_value(), "the chunk form takes a status word");
        same_device(in, *status, "status");
        want(*status, torch::kInt32, "status");
        const uintptr_t at = reinterpret_cast<uintptr_t>(workspace->data_ptr()), first = (at + 1023) & ~(uintptr_t)1023;
        TORCH_CHECK(workspace->numel() >= (int64_t)(first - at + llm::gdn_chunk_bytes(1, p.n_k, p.n_v)), "workspace too small");
        check(llm::launch_gdn_chunk(p, reinterpret_cast<void*>(first), workspace->numel() - (first - at), status->data_ptr<int>(), launches, stream()), "gdn_prefill");
    } else {
        check(llm::launch_gdn_rows(p, stream()), "gdn_prefill");
    }
    check(llm::launch_gdn_windows(p, stream()), "gdn_prefill");
    return launches + 1;
}

// keep: decays [B, R, n_v], keys and corrections [B, R, n_v, d], convolution inputs [B, R, C]
void keep_args(llm::GdnParams& p, const Tensor& like, const std::vector<Tensor>& keep) {
    TORCH_CHECK(keep.size() == 4 && keep[3].dim() == 3, "keep");
    const int64_t B = p.n_seqs, R = keep[3].size(1), n = B * R * p.n_v;
    TORCH_CHECK(keep[3].size(0) == B && keep[3].size(2) == p.C, "kept rows of other sizes");
    p.rows_per_seq = R;
    p.keep_a = const_cast<float*>(floats_on(like, keep[0], n, "decays")); p.keep_k = const_cast<float*>(floats_on(like, keep[1], n * p.d, "keys"));
    p.keep_u = const_cast<float*>(floats_on(like, keep[2], n * p.d, "corrections"));
    TORCH_CHECK(((reinterpret_cast<uintptr_t>(p.keep_k) | reinterpret_cast<uintptr_t>(p.keep_u)) & 15) == 0, "keys and corrections must start on 16 bytes");
    same_device(like, keep[3], "inputs");
    want(keep[3], torch::kBFloat16, "inputs");
    p.keep_x = reinterpret_cast<__nv_bfloat16*>(keep[3].data_ptr());
}

int gdn_verify(const Tensor& in, int64_t C, int64_t z_off, int64_t ab_off, const Tensor& conv_w, const Tensor& ssm_a, const Tensor& dt_bias, const Tensor& norm_w,
               const Tensor& conv, const Tensor& rec, const Tensor& slots, const Tensor& out, int64_t n_k, int64_t v_head_offset, double eps, const std::vector<Tensor>& keep,
               const Tensor& status) {
    llm::GdnParams p = gdn_params(in, C, z_off, ab_off, conv_w, ssm_a, dt_bias, norm_w, conv, rec, slots, out, n_k, v_head_offset, eps);
    keep_args(p, in, keep);
    TORCH_CHECK(in.size(0) == (int64_t)p.n_seqs * p.rows_per_seq, "in must have the same number of rows for every sequence");
    same_device(in, status, "status");
    want(status, torch::kInt32, "status");
    p.status = status.data_ptr<int>();
    const c10::cuda::CUDAGuard guard(in.device());
    check(llm::launch_gdn_rows(p, stream()), "gdn_verify");
    return 1;
}

void gdn_commit(const std::vector<Tensor>& keep, const Tensor& accepted, const Tensor& conv, const Tensor& rec, const Tensor& slots, int64_t n_k) {
    llm::GdnParams p = gdn_state(conv, rec, n_k);
    p.n_seqs = slots.numel();
    TORCH_CHECK(p.n_seqs <= 65535, "more than 65535 sequences");
    p.slots = ints_on(rec, slots, p.n_seqs, "slots");
    keep_args(p, rec, keep);
    const int* n = ints_on(rec, accepted, p.n_seqs, "n_rows");
    const c10::cuda::CUDAGuard guard(rec.device());
    check(llm::launch_gdn_commit(p, n, stream()), "gdn_commit");
}

// A layer of the paged cache, bf16 or (`q8`) 8-bit
void cache_args(const Tensor& like, const Tensor& kv, int64_t kv_heads, int64_t head_dim, uint8_t*& at, int& n_pages, size_t& page_bytes, size_t& scale_off, int& q8) {
    same_device(like, kv, "kv");
    TORCH_CHECK(kv.is_contiguous() && reinterpret_cast<uintptr_t>(kv.data_ptr()) % 16 == 0, "kv must be contiguous and 16-byte aligned");
    scale_off = (size_t)2 * kv_heads * 64 * head_dim;
    q8 = kv.scalar_type() == torch::kUInt8;
    if (q8) {
        page_bytes = scale_off + scale_off / 16;
        TORCH_CHECK(kv.dim() == 2 && (size_t)kv.size(1) == page_bytes, "an 8-bit cache layer is [n_pages, bytes of a page of these heads]");
    } else {
        page_bytes = 2 * scale_off;
        TORCH_CHECK(kv.scalar_type() == torch::kBFloat16, "the cache must be bf16 or 8-bit");
        TORCH_CHECK(kv.dim() == 5 && kv.size(1) == 2 && kv.size(2) == kv_heads && kv.size(3) == 64 && kv.size(4) == head_dim, "a cache layer is [n_pages, 2, kv heads, 64, head size]");
    }
    at = static_cast<uint8_t*>(kv.data_ptr()); n_pages = kv.size(0);
}
const int* table_arg(const Tensor& like, const Tensor& t, int& n_seqs, int& max_pages) {
    same_device(like, t, "block_table");
    TORCH_CHECK(t.dim() == 2, "block_table must be [sequences, pages]");
    n_seqs = t.size(0); max_pages = t.size(1);
    return ints(t, "block_table");
}

void rope_part_kv(const Tensor& rows, const Tensor& q_out, const Tensor& kv, const OptTensor& q_norm, const OptTensor& k_norm, const Tensor& freqs, double magnitude,
                  const Tensor& positions, const Tensor& seq_ids, const Tensor& block_table, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, double eps, bool gated, bool interleaved) {
    llm::RopePartParams p = {};
    p.rows = bf16_rows(rows, "rows");
    TORCH_CHECK(head_dim == 64 || head_dim == 128 || head_dim == 256, "head size must be 64, 128 or 256");
    TORCH_CHECK(n_heads >= 1 && n_kv_heads >= 1 && n_heads <= 4096 && n_kv_heads <= 4096, "heads");
    TORCH_CHECK(rows.size(1) == (n_heads * (gated ? 2 : 1) + 2 * n_kv_heads) * head_dim, "rows must be [query (and gate) per head | keys | values]");
    const int64_t T = rows.size(0), lane = head_dim / 32;
    TORCH_CHECK(T <= INT32_MAX, "too many rows");
    p.row = rows.stride(0); p.q_stride = (gated ? 2 : 1) * head_dim;
    p.whole = reinterpret_cast<uintptr_t>(rows.data_ptr()) % (2 * lane) == 0 && (T <= 1 || rows.stride(0) % lane == 0);
    if (q_norm) p.q_norm = floats_on(rows, *q_norm, head_dim, "q_norm");
    if (k_norm) p.k_norm = floats_on(rows, *k_norm, head_dim, "k_norm");
    same_device(rows, freqs, "freqs");
    want(freqs, torch::kFloat64, "freqs");
    TORCH_CHECK(freqs.numel() * 2 <= head_dim, "more frequencies than a head has pairs");
    p.freqs = freqs.data_ptr<double>(); p.rot = 2 * freqs.numel(); p.magnitude = magnitude; p.interleaved = interleaved;
    p.positions = ints_on(rows, positions, T, "positions"); p.seq_ids = ints_on(rows, seq_ids, T, "seq_ids");
    p.block_table = table_arg(rows, block_table, p.n_seqs, p.max_pages);
    p.n_tokens = T; p.n_heads = n_heads; p.n_kv_heads = n_kv_heads; p.head_dim = head_dim; p.eps = eps;
    same_device(rows, q_out, "q_out");
    want(q_out, torch::kBFloat16, "q_out");
    TORCH_CHECK(q_out.numel() == T * n_heads * head_dim && reinterpret_cast<uintptr_t>(q_out.data_ptr()) % 16 == 0, "q_out must be [rows, heads, head size], 16-byte aligned");
    p.q_out = reinterpret_cast<__nv_bfloat16*>(q_out.data_ptr());
    cache_args(rows, kv, n_kv_heads, head_dim, p.kv, p.n_pages, p.page_bytes, p.scale_off, p.q8);
    const c10::cuda::CUDAGuard guard(rows.device());
    check(llm::launch_rope_part(p, stream()), "rope_part_kv");
}

// Returns the number of launches
int attn_decode_shared(const Tensor& q, const Tensor& kv, const Tensor& out, const Tensor& block_table, const Tensor& seq_lens, const Tensor& shared_len, int64_t n_heads, int64_t n_kv_heads,
                       int64_t head_dim, int64_t rows_per_seq, double scale, const OptTensor& gate, int64_t max_shared, int64_t max_tail, int64_t prefix_row, const Tensor& tickets, const Tensor& status) {
    llm::AttnSharedParams p = {};
    want(q, torch::kBFloat16, "q");
    TORCH_CHECK(head_dim == 64 || head_dim == 128 || head_dim == 256, "head size must be 64, 128 or 256");
    TORCH_CHECK(n_kv_heads >= 1 && n_heads >= 1 && n_heads <= 65535 && n_heads % n_kv_heads == 0, "query heads must be a multiple of K/V heads");
    TORCH_CHECK(rows_per_seq >= 1 && n_heads / n_kv_heads * rows_per_seq <= 16, "at most 16 rows x heads of a group per sequence");
    TORCH_CHECK((float)scale > 0.f && scale <= FLT_MAX, "scale must be positive and finite");
    p.block_table = table_arg(q, block_table, p.n_seqs, p.max_pages);
    TORCH_CHECK(p.n_seqs <= 65535 && (int64_t)p.max_pages * 64 <= INT32_MAX, "more than 65535 sequences, or too many pages");
    TORCH_CHECK(q.numel() == p.n_seqs * rows_per_seq * n_heads * head_dim, "q must be [sequences * rows, heads, head size]");
    same_device(q, out, "out");
    want(out, torch::kBFloat16, "out");
    TORCH_CHECK(out.numel() == q.numel(), "out must be like q");
    TORCH_CHECK(((reinterpret_cast<uintptr_t>(q.data_ptr()) | reinterpret_cast<uintptr_t>(out.data_ptr())) & 15) == 0, "q and out must be 16-byte aligned");
    uint8_t* at = nullptr;
    size_t page_bytes = 0, scale_off = 0;
    int q8 = 0;
    cache_args(q, kv, n_kv_heads, head_dim, at, p.n_pages, page_bytes, scale_off, q8);
    TORCH_CHECK(!q8, "attention behind a shared prefix reads bf16 pages");
    p.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr()); p.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr()); p.kv = reinterpret_cast<const __nv_bfloat16*>(at);
    p.seq_lens = ints_on(q, seq_lens, p.n_seqs, "seq_lens");
    p.shared_len = ints_on(q, shared_len, 1, "shared_len");
    p.rows_per_seq = rows_per_seq; p.n_heads = n_heads; p.n_kv_heads = n_kv_heads; p.head_dim = head_dim; p.scale = scale;
    if (gate) {
        same_device(q, *gate, "gate");
        TORCH_CHECK(gate->scalar_type() == torch::kBFloat16 && gate->dim() == 3 && gate->size(0) == p.n_seqs * rows_per_seq && gate->size(1) == n_heads && gate->size(2) == head_dim && gate->stride(2) == 1 &&
                    gate->stride(0) >= 0 && gate->stride(1) >= 0, "gate must be bf16 [rows, heads, head size]");
        p.gate = reinterpret_cast<const __nv_bfloat16*>(gate->data_ptr()); p.gate_token = gate->stride(0); p.gate_head = gate->stride(1);
    }
    TORCH_CHECK(max_shared >= 0 && max_tail >= 0 && prefix_row >= 0 && (p.n_seqs == 0 || prefix_row < p.n_seqs), "max_shared, max_tail or prefix_row");
    if (p.n_seqs == 0) return 0;
    const int64_t table = (int64_t)p.max_pages * 64;
    p.prefix_row = prefix_row;
    same_device(q, tickets, "tickets"); same_device(q, status, "status");
    want(status, torch::kInt32, "status");
    const int* t = ints(tickets, "tickets");
    const int64_t most = std::min(max_shared, table), rest = std::max<int64_t>(table - most, 64);
    const llm::AttnSharedPlan plan = llm::attn_shared_plan(p.n_seqs, p.rows_per_seq, p.n_heads, p.n_kv_heads, p.head_dim, most, max_tail ? std::min(max_tail, table) : rest, tickets.numel());
    const c10::cuda::CUDAGuard guard(q.device());
    p.splits = plan.splits; p.tail_splits = plan.tail_splits; p.tickets = reinterpret_cast<unsigned*>(const_cast<int*>(t));
    const int64_t rows = plan.prefix_rows + plan.tail_rows;
    Tensor parts;
    if (rows) {
        parts = torch::empty({rows * (head_dim + 2)}, q.options().dtype(torch::kFloat32));
        p.part_o = parts.data_ptr<float>(); p.tail_o = p.part_o + plan.prefix_rows * head_dim;
        p.part_ml = p.part_o + rows * head_dim; p.tail_ml = p.part_ml + plan.prefix_rows * 2;
    }
    check(llm::launch_attn_shared(p, status.data_ptr<int>(), stream()), "attn_decode_shared");
    return p.splits ? 2 : 1;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("gdn_prefill", &gdn_prefill);
    m.def("gdn_verify", &gdn_verify);
    m.def("gdn_commit", &gdn_commit);
    m.def("gdn_chunk_bytes", &llm::gdn_chunk_bytes);
    m.def("rope_part_kv", &rope_part_kv);
    m.def("attn_decode_shared", &attn_decode_shared);
    m.def("set_pdl", [](bool on) { llm::pdl_enabled() = on; });
    m.def("bounds_status", [](bool reset) { return llm::bounds_status_gdn_rows(reset) | llm::bounds_status_gdn_chunk(reset) | llm::bounds_status_rope_part(reset) | llm::bounds_status_attn_shared(reset); });
}
