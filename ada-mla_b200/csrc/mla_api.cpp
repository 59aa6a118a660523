// mla_api.cpp -- PyTorch extension boundary, mirroring the reference's
// csrc/mla_api.cpp (PYBIND11_MODULE(ada_mla), :115-120): the same three names
// with the same (query, cache) -> Tensor signatures, output shapes and dtypes,
// plus the batched/varlen entry point and the LSE merge used by the
// multi-GPU layer.  Every function validates device / dtype / contiguity /
// shape, allocates outputs and workspace from the caching allocator, and calls
// the C ABI (include/mla_b200.h) on the current torch stream; a non-zero status
// raises.  No torch types cross the C ABI.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "mla_b200.h"

namespace {

void check_status(int st, const char *what) {
    if (st == MLA_B200_ERR_CUDA) {
        const auto e = static_cast<cudaError_t>(mla_b200_last_cuda_error());
        TORCH_CHECK(false, what, " failed: ", mla_b200_status_string(st), " (status ", st, ", ",
                    cudaGetErrorName(e), ")");
    }
    TORCH_CHECK(st == MLA_B200_OK, what, " failed: ", mla_b200_status_string(st), " (status ", st,
                ")");
}

void check_cuda(const at::Tensor &t, const char *name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

void *stream_ptr() { return static_cast<void *>(at::cuda::getCurrentCUDAStream().stream()); }

// An uninitialised tensor straight from the caching allocator (at::empty without its
// dispatch: about a microsecond less, which is what a step of small calls is made of).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor &like) {
    return at::Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt));
}

// Tensors that share one allocation, each at a multiple of 16 bytes.
class Carve {
  public:
    Carve(int64_t bytes, const at::Tensor &like) : base_(fresh({std::max<int64_t>(bytes, 16)}, at::kByte, like)) {}
    static int64_t room(int64_t n, int64_t size) { return (n * size + 15) / 16 * 16; }
    at::Tensor take(int64_t n, at::ScalarType dtype) {
        const int64_t size = c10::elementSize(dtype);
        auto t = c10::make_intrusive<c10::TensorImpl>(c10::Storage(base_.storage()), base_.key_set(),
                                                      c10::scalarTypeToTypeMeta(dtype));
        t->set_storage_offset(at_ / size);
        t->set_sizes_contiguous({n});
        at_ += room(n, size);
        return at::Tensor(std::move(t));
    }

  private:
    at::Tensor base_;
    int64_t at_ = 0;
};

at::Tensor workspace(const at::Tensor &like, size_t bytes) {
    return at::empty({(int64_t)std::max<size_t>(bytes, 256)},
                     at::TensorOptions().device(like.device()).dtype(at::kByte));
}

}  // namespace

// Reference: mla_decode_naive (csrc/mla_api.cpp:5-32).  fp32, scale
// 1/sqrt(head_dim_c), returns all head_dim_c columns: [n_h, head_dim_c].
at::Tensor mla_decode_naive(const at::Tensor &query, const at::Tensor &cache) {
    check_cuda(query, "query");
    check_cuda(cache, "cache");
    TORCH_CHECK(query.scalar_type() == at::kFloat && cache.scalar_type() == at::kFloat,
                "mla_decode_naive: query and cache must be float32");
    TORCH_CHECK(query.dim() == 2 && cache.dim() == 2 && query.size(1) == cache.size(1),
                "mla_decode_naive: expected query [n_h, D] and cache [N, D]");
    TORCH_CHECK(cache.size(0) > 0, "mla_decode_naive: empty cache");
    TORCH_CHECK(query.device() == cache.device(), "query and cache on different devices");
    c10::cuda::CUDAGuard g(query.device());
    const int64_t nh = query.size(0), d = query.size(1), n = cache.size(0);
    at::Tensor out = at::empty({nh, d}, query.options());
    at::Tensor attn = at::empty({nh, n}, query.options());
    check_status(mla_b200_decode_naive_f32(query.data_ptr<float>(), cache.data_ptr<float>(),
                                           attn.data_ptr<float>(), out.data_ptr<float>(), (int)nh,
                                           (int)d, (int)n, stream_ptr()),
                 "mla_decode_naive");
    return out;
}

static at::Tensor fused_f32(const at::Tensor &query, const at::Tensor &cache) {
    const int64_t nh = query.size(0), n = cache.size(0);
    at::Tensor out = at::empty({nh, MLA_B200_HEAD_DIM_V}, query.options());
    const size_t ws = mla_b200_workspace_size(1, (int)nh, n, (int)n, 0);
    at::Tensor w = workspace(query, ws);
    check_status(mla_b200_decode_fused_f32(query.data_ptr<float>(), cache.data_ptr<float>(),
                                           out.data_ptr<float>(), (int)nh,
                                           (int)query.size(1), (int)n, w.data_ptr(), w.numel(),
                                           stream_ptr()),
                 "mla_decode_fused");
    return out;
}

static void check_decode_inputs(const at::Tensor &query, const at::Tensor &cache, const char *fn) {
    check_cuda(query, "query");
    check_cuda(cache, "cache");
    TORCH_CHECK(query.device() == cache.device(), fn, ": query and cache on different devices");
    TORCH_CHECK(query.dim() == 2 && query.size(1) == MLA_B200_HEAD_DIM_K, fn,
                ": query must be [n_h, 576]");
    TORCH_CHECK(cache.dim() == 2 && cache.size(1) == MLA_B200_HEAD_DIM_K, fn,
                ": cache must be [N, 576]");
    TORCH_CHECK(query.scalar_type() == cache.scalar_type(), fn,
                ": query and cache must have the same dtype");
}

// Reference: mla_decode_fused (csrc/mla_api.cpp:34-54).  fp32 in, fp32
// [n_h, 512] out, scale 1/sqrt(192).
at::Tensor mla_decode_fused(const at::Tensor &query, const at::Tensor &cache) {
    check_decode_inputs(query, cache, "mla_decode_fused");
    TORCH_CHECK(query.scalar_type() == at::kFloat, "mla_decode_fused: float32 inputs expected");
    c10::cuda::CUDAGuard g(query.device());
    return fused_f32(query, cache);
}

// Reference: mla_decode_split (csrc/mla_api.cpp:86-113).  fp16 -> the split-KV
// decode, [n_h, 512] fp16; fp32 -> the fp32 kernel (the reference's fp32
// specialization is an empty stub, csrc/mla_decode_splitk_fwd_sm89.cu:9-24).
// num_splits <= 0 selects the heuristic (the reference hard-codes 4).
at::Tensor mla_decode_split(const at::Tensor &query, const at::Tensor &cache, int64_t num_splits) {
    check_decode_inputs(query, cache, "mla_decode_split");
    c10::cuda::CUDAGuard g(query.device());
    if (query.scalar_type() == at::kFloat) return fused_f32(query, cache);
    TORCH_CHECK(query.scalar_type() == at::kHalf,
                "mla_decode_split: float16 or float32 inputs expected");
    const int64_t nh = query.size(0), n = cache.size(0);
    at::Tensor out = at::empty({nh, MLA_B200_HEAD_DIM_V}, query.options());
    const size_t ws = mla_b200_workspace_size(1, (int)nh, n, (int)n, (int)num_splits);
    at::Tensor w = workspace(query, ws);
    check_status(mla_b200_decode_split_f16(query.data_ptr(), cache.data_ptr(), out.data_ptr(),
                                           (int)nh, (int)n, (int)num_splits, w.data_ptr(),
                                           w.numel(), stream_ptr()),
                 "mla_decode_split");
    return out;
}

// Batched / varlen decode (no reference counterpart).
//   query [B, n_h, 576] fp16 or bf16 (cache the same dtype); cache [B, N, 576]
//   (dense) or [T, 576] with cu_seqlens int32 [B+1] on the same device (packed).
// Returns (out [B, n_h, 512] in the input dtype, or fp32 when out_fp32,
// lse [B, n_h] fp32 or empty).
std::vector<at::Tensor> mla_decode_batched(const at::Tensor &query, const at::Tensor &cache,
                                           const c10::optional<at::Tensor> &cu_seqlens,
                                           int64_t max_seq_len, double softmax_scale,
                                           int64_t num_splits, bool return_lse,
                                           bool out_fp32, double kv_scale) {
    check_cuda(query, "query");
    check_cuda(cache, "cache");
    TORCH_CHECK(query.device() == cache.device(), "query and cache on different devices");
    const bool bf16 = query.scalar_type() == at::kBFloat16;
    const bool fp8 = cache.scalar_type() == at::kFloat8_e4m3fn;
    TORCH_CHECK((query.scalar_type() == at::kHalf || bf16) &&
                    (cache.scalar_type() == query.scalar_type() || (fp8 && !bf16)),
                "mla_decode_batched: float16 or bfloat16 inputs (query and cache alike), or a "
                "float16 query with a float8_e4m3fn cache, expected");
    TORCH_CHECK(query.dim() == 3 && query.size(2) == MLA_B200_HEAD_DIM_K,
                "mla_decode_batched: query must be [B, n_h, 576]");
    const int64_t b = query.size(0), nh = query.size(1);
    c10::cuda::CUDAGuard g(query.device());
    const int32_t *cu_ptr = nullptr;
    int64_t total = 0;
    if (cu_seqlens.has_value() && cu_seqlens->defined()) {
        const at::Tensor &cu = *cu_seqlens;
        check_cuda(cu, "cu_seqlens");
        TORCH_CHECK(cu.device() == query.device(), "cu_seqlens on a different device");
        TORCH_CHECK(cu.scalar_type() == at::kInt && cu.dim() == 1 && cu.size(0) == b + 1,
                    "cu_seqlens must be int32 [B+1]");
        TORCH_CHECK(cache.dim() == 2 && cache.size(1) == MLA_B200_HEAD_DIM_K,
                    "packed cache must be [T, 576]");
        total = cache.size(0);
        if (max_seq_len < 0) {
            max_seq_len = b > 0 ? (cu.slice(0, 1) - cu.slice(0, 0, b)).max().item<int64_t>() : 0;
        }
        cu_ptr = cu.data_ptr<int32_t>();
    } else {
        TORCH_CHECK(cache.dim() == 3 && cache.size(0) == b && cache.size(2) == MLA_B200_HEAD_DIM_K,
                    "dense cache must be [B, N, 576]");
        max_seq_len = cache.size(1);
        total = b * max_seq_len;
    }
    at::Tensor out = at::empty({b, nh, MLA_B200_HEAD_DIM_V},
                               query.options().dtype(out_fp32 ? at::kFloat
                                                              : query.scalar_type()));
    at::Tensor lse = return_lse ? at::empty({b, nh}, query.options().dtype(at::kFloat))
                                : at::Tensor();
    const size_t ws = (fp8 ? mla_b200_workspace_size_fp8 : mla_b200_workspace_size)(
        (int)b, (int)nh, total, (int)max_seq_len, (int)num_splits);
    at::Tensor w = workspace(query, ws);
    const int odt = out_fp32 ? MLA_B200_OUT_F32 : (bf16 ? MLA_B200_OUT_BF16 : MLA_B200_OUT_F16);
    float *lse_ptr = return_lse ? lse.data_ptr<float>() : nullptr;
    if (fp8) {
        check_status(mla_b200_decode_batched_fp8(
                         query.data_ptr(), cache.data_ptr(), (float)kv_scale, cu_ptr, (int)b, (int)nh,
                         total, (int)max_seq_len, (float)softmax_scale, (int)num_splits,
                         out.data_ptr(), odt, lse_ptr, w.data_ptr(), w.numel(), stream_ptr()),
                     "mla_decode_batched");
    } else {
        auto *fn = bf16 ? mla_b200_decode_batched_bf16 : mla_b200_decode_batched_f16;
        check_status(fn(query.data_ptr(), cache.data_ptr(), cu_ptr, (int)b, (int)nh, total,
                        (int)max_seq_len, (float)softmax_scale, (int)num_splits, out.data_ptr(), odt,
                        lse_ptr, w.data_ptr(), w.numel(), stream_ptr()),
                     "mla_decode_batched");
    }
    if (!return_lse) lse = at::empty({0}, query.options().dtype(at::kFloat));
    return {out, lse};
}

// Multi-token decode (no reference counterpart).
//   query [B, k, n_h, 576] fp16 or bf16 (n_h <= 128), cache as in
//   mla_decode_batched (same dtype); draft token i of sequence b sees its first
//   len_b - (k - 1 - i) tokens.  Returns (out [B, k, n_h, 512], lse [B, k, n_h] or empty).
std::vector<at::Tensor> mla_decode_mtp(const at::Tensor &query, const at::Tensor &cache,
                                       const c10::optional<at::Tensor> &cu_seqlens,
                                       int64_t max_seq_len, double softmax_scale,
                                       int64_t num_splits, bool return_lse, bool out_fp32) {
    check_cuda(query, "query");
    check_cuda(cache, "cache");
    TORCH_CHECK(query.device() == cache.device(), "query and cache on different devices");
    const bool bf16 = query.scalar_type() == at::kBFloat16;
    TORCH_CHECK((query.scalar_type() == at::kHalf || bf16) && cache.scalar_type() == query.scalar_type(),
                "mla_decode_mtp: float16 or bfloat16 inputs (query and cache alike) expected");
    TORCH_CHECK(query.dim() == 4 && query.size(3) == MLA_B200_HEAD_DIM_K,
                "mla_decode_mtp: query must be [B, k, n_h, 576]");
    const int64_t b = query.size(0), k = query.size(1), nh = query.size(2);
    c10::cuda::CUDAGuard g(query.device());
    const int32_t *cu_ptr = nullptr;
    int64_t total = 0;
    if (cu_seqlens.has_value() && cu_seqlens->defined()) {
        const at::Tensor &cu = *cu_seqlens;
        check_cuda(cu, "cu_seqlens");
        TORCH_CHECK(cu.device() == query.device(), "cu_seqlens on a different device");
        TORCH_CHECK(cu.scalar_type() == at::kInt && cu.dim() == 1 && cu.size(0) == b + 1,
                    "cu_seqlens must be int32 [B+1]");
        TORCH_CHECK(cache.dim() == 2 && cache.size(1) == MLA_B200_HEAD_DIM_K,
                    "packed cache must be [T, 576]");
        total = cache.size(0);
        if (max_seq_len < 0)
            max_seq_len = b > 0 ? (cu.slice(0, 1) - cu.slice(0, 0, b)).max().item<int64_t>() : 0;
        cu_ptr = cu.data_ptr<int32_t>();
    } else {
        TORCH_CHECK(cache.dim() == 3 && cache.size(0) == b && cache.size(2) == MLA_B200_HEAD_DIM_K,
                    "dense cache must be [B, N, 576]");
        max_seq_len = cache.size(1);
        total = b * max_seq_len;
    }
    at::Tensor out = at::empty({b, k, nh, MLA_B200_HEAD_DIM_V},
                               query.options().dtype(out_fp32 ? at::kFloat : query.scalar_type()));
    at::Tensor lse = return_lse ? at::empty({b, k, nh}, query.options().dtype(at::kFloat)) : at::Tensor();
    const size_t ws = mla_b200_workspace_size_mtp((int)b, (int)k, (int)nh, total, (int)max_seq_len,
                                                  (int)num_splits);
    at::Tensor w = workspace(query, ws);
    auto *fn = bf16 ? mla_b200_decode_mtp_bf16 : mla_b200_decode_mtp_f16;
    const int odt = out_fp32 ? MLA_B200_OUT_F32 : (bf16 ? MLA_B200_OUT_BF16 : MLA_B200_OUT_F16);
    check_status(fn(query.data_ptr(), cache.data_ptr(), cu_ptr, (int)b, (int)k, (int)nh, total,
                    (int)max_seq_len, (float)softmax_scale, (int)num_splits, out.data_ptr(), odt,
                    return_lse ? lse.data_ptr<float>() : nullptr, w.data_ptr(), w.numel(),
                    stream_ptr()),
                 "mla_decode_mtp");
    if (!return_lse) lse = at::empty({0}, query.options().dtype(at::kFloat));
    return {out, lse};
}

// Paged decode (no reference counterpart).
//   query [B, n_h, 576] fp16 or bf16; kv_pages [num_pages, page_size, 576] in the
//   same dtype; block_table int32 [B, max_blocks]; seq_lens int32 [B]; all on
//   one device.  max_seq_len < 0 reads max(seq_lens) from the device.
// Returns (out [B, n_h, 512] in the input dtype or fp32, lse [B, n_h] fp32 or empty).
std::vector<at::Tensor> mla_decode_paged(const at::Tensor &query, const at::Tensor &kv_pages,
                                         const at::Tensor &block_table, const at::Tensor &seq_lens,
                                         int64_t max_seq_len, double softmax_scale,
                                         int64_t num_splits, bool return_lse, bool out_fp32) {
    check_cuda(query, "query");
    check_cuda(kv_pages, "kv_pages");
    check_cuda(block_table, "block_table");
    check_cuda(seq_lens, "seq_lens");
    TORCH_CHECK(query.device() == kv_pages.device() && query.device() == block_table.device() &&
                    query.device() == seq_lens.device(),
                "mla_decode_paged: all tensors on one device");
    const bool bf16 = query.scalar_type() == at::kBFloat16;
    TORCH_CHECK((query.scalar_type() == at::kHalf || bf16) &&
                    kv_pages.scalar_type() == query.scalar_type(),
                "mla_decode_paged: float16 or bfloat16 inputs (query and kv_pages alike) expected");
    TORCH_CHECK(query.dim() == 3 && query.size(2) == MLA_B200_HEAD_DIM_K,
                "mla_decode_paged: query must be [B, n_h, 576]");
    TORCH_CHECK(kv_pages.dim() == 3 && kv_pages.size(2) == MLA_B200_HEAD_DIM_K,
                "mla_decode_paged: kv_pages must be [num_pages, page_size, 576]");
    const int64_t b = query.size(0), nh = query.size(1);
    TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 &&
                    block_table.size(0) == b,
                "mla_decode_paged: block_table must be int32 [B, max_blocks]");
    TORCH_CHECK(seq_lens.scalar_type() == at::kInt && seq_lens.dim() == 1 && seq_lens.size(0) == b,
                "mla_decode_paged: seq_lens must be int32 [B]");
    c10::cuda::CUDAGuard g(query.device());
    const int64_t num_pages = kv_pages.size(0), page_size = kv_pages.size(1);
    const int64_t max_blocks = block_table.size(1);
    if (max_seq_len < 0) max_seq_len = b > 0 ? seq_lens.max().item<int64_t>() : 0;
    at::Tensor out = at::empty({b, nh, MLA_B200_HEAD_DIM_V},
                               query.options().dtype(out_fp32 ? at::kFloat
                                                              : query.scalar_type()));
    at::Tensor lse = return_lse ? at::empty({b, nh}, query.options().dtype(at::kFloat))
                                : at::Tensor();
    const size_t ws = mla_b200_workspace_size((int)b, (int)nh, b * max_seq_len, (int)max_seq_len,
                                              (int)num_splits);
    at::Tensor w = workspace(query, ws);
    auto *fn = bf16 ? mla_b200_decode_paged_bf16 : mla_b200_decode_paged_f16;
    const int odt = out_fp32 ? MLA_B200_OUT_F32 : (bf16 ? MLA_B200_OUT_BF16 : MLA_B200_OUT_F16);
    check_status(fn(query.data_ptr(), kv_pages.data_ptr(), block_table.data_ptr<int32_t>(),
                    seq_lens.data_ptr<int32_t>(), (int)b, (int)nh, (int)num_pages, (int)page_size,
                    (int)max_blocks, (int)max_seq_len, (float)softmax_scale, (int)num_splits,
                    out.data_ptr(), odt, return_lse ? lse.data_ptr<float>() : nullptr,
                    w.data_ptr(), w.numel(), stream_ptr()),
                 "mla_decode_paged");
    if (!return_lse) lse = at::empty({0}, query.options().dtype(at::kFloat));
    return {out, lse};
}

// Draft-tree decode over a paged cache (no reference counterpart).
//   query [B, k, n_h, 576] fp16 or bf16 (k <= 64, n_h <= 128); kv_pages [num_pages,
//   page_size, 576] in the same dtype; block_table int32 [B, max_blocks]; seq_lens
//   int32 [B]; tree_mask int64 [B, k] or [k] (bit j of draft i's word: i sees draft
//   j), or None for a chain.  max_seq_len < 0 reads max(seq_lens) from the device.
// Returns (out [B, k, n_h, 512], lse [B, k, n_h] fp32 or empty).
std::vector<at::Tensor> mla_decode_tree(const at::Tensor &query, const at::Tensor &kv_pages,
                                        const at::Tensor &block_table, const at::Tensor &seq_lens,
                                        const c10::optional<at::Tensor> &tree_mask, int64_t max_seq_len,
                                        double softmax_scale, int64_t num_splits, bool return_lse,
                                        bool out_fp32) {
    check_cuda(query, "query");
    check_cuda(kv_pages, "kv_pages");
    check_cuda(block_table, "block_table");
    check_cuda(seq_lens, "seq_lens");
    const bool bf16 = query.scalar_type() == at::kBFloat16;
    TORCH_CHECK((query.scalar_type() == at::kHalf || bf16) && kv_pages.scalar_type() == query.scalar_type(),
                "mla_decode_tree: float16 or bfloat16 inputs (query and kv_pages alike) expected");
    TORCH_CHECK(query.dim() == 4 && query.size(3) == MLA_B200_HEAD_DIM_K,
                "mla_decode_tree: query must be [B, k, n_h, 576]");
    TORCH_CHECK(kv_pages.dim() == 3 && kv_pages.size(2) == MLA_B200_HEAD_DIM_K,
                "mla_decode_tree: kv_pages must be [num_pages, page_size, 576]");
    const int64_t b = query.size(0), k = query.size(1), nh = query.size(2);
    TORCH_CHECK(k >= 1 && k <= 64, "mla_decode_tree: 1 to 64 drafts expected");
    TORCH_CHECK(nh >= 1 && nh <= 128, "mla_decode_tree: 1 to 128 heads expected");
    TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == b,
                "mla_decode_tree: block_table must be int32 [B, max_blocks]");
    TORCH_CHECK(seq_lens.scalar_type() == at::kInt && seq_lens.dim() == 1 && seq_lens.size(0) == b,
                "mla_decode_tree: seq_lens must be int32 [B]");
    TORCH_CHECK(query.device() == kv_pages.device() && query.device() == block_table.device() &&
                    query.device() == seq_lens.device(),
                "mla_decode_tree: all tensors on one device");
    const uint64_t *mask = nullptr;
    int shared = 0;
    if (tree_mask.has_value() && tree_mask->defined()) {
        const at::Tensor &m = *tree_mask;
        check_cuda(m, "tree_mask");
        shared = m.dim() == 1;
        TORCH_CHECK(m.scalar_type() == at::kLong && m.device() == query.device() &&
                        ((shared && m.size(0) == k) || (m.dim() == 2 && m.size(0) == b && m.size(1) == k)),
                    "mla_decode_tree: tree_mask must be int64 [B, k] or [k] on the query's device");
        mask = reinterpret_cast<const uint64_t *>(m.data_ptr<int64_t>());
    }
    c10::cuda::CUDAGuard g(query.device());
    if (max_seq_len < 0) max_seq_len = b > 0 ? std::max<int64_t>(seq_lens.max().item<int64_t>(), 0) : 0;
    TORCH_CHECK(max_seq_len <= INT32_MAX, "mla_decode_tree: max_seq_len out of range");
    at::Tensor out = fresh({b, k, nh, MLA_B200_HEAD_DIM_V}, out_fp32 ? at::kFloat : query.scalar_type(), query);
    at::Tensor lse = fresh({return_lse ? b : 0, k, nh}, at::kFloat, query);
    at::Tensor w = fresh({(int64_t)std::max<size_t>(mla_b200_workspace_size_tree((int)b, (int)k, (int)nh, (int)max_seq_len,
                                                                                (int)num_splits), 256)},
                         at::kByte, query);
    auto *fn = bf16 ? mla_b200_decode_tree_bf16 : mla_b200_decode_tree_f16;
    const int odt = out_fp32 ? MLA_B200_OUT_F32 : (bf16 ? MLA_B200_OUT_BF16 : MLA_B200_OUT_F16);
    check_status(fn(query.data_ptr(), kv_pages.data_ptr(), block_table.data_ptr<int32_t>(),
                    seq_lens.data_ptr<int32_t>(), mask, shared, (int)b, (int)k, (int)nh, (int)kv_pages.size(0),
                    (int)kv_pages.size(1), (int)block_table.size(1), (int)max_seq_len, (float)softmax_scale,
                    (int)num_splits, out.data_ptr(), odt, return_lse ? lse.data_ptr<float>() : nullptr,
                    w.data_ptr(), w.numel(), stream_ptr()),
                 "mla_decode_tree");
    return {out, lse};
}

// Attention over prompts in expanded form (no reference counterpart).
//   query [Tq, n_h, 192], k_nope and v [Tk, n_h, 128], k_rope [Tk, 64], fp16 or bf16
//   alike, packed by int32 cu_seqlens_q / cu_seqlens_k [B + 1]; or, without them,
//   [B, Lq, n_h, 192], [B, Lk, n_h, 128], [B, Lk, 64].  Any strides with a dense last
//   dimension and 16-byte multiples; dense sequences of more than one row follow one
//   another.  max_seq_len_* < 0 reads them from the device.
// Returns (out [.., n_h, 128], lse [.., n_h] fp32 or empty).
std::vector<at::Tensor> mla_prefill(const at::Tensor &query, const at::Tensor &k_nope, const at::Tensor &k_rope,
                                    const at::Tensor &v, const c10::optional<at::Tensor> &cu_seqlens_q,
                                    const c10::optional<at::Tensor> &cu_seqlens_k, int64_t max_seq_len_q,
                                    int64_t max_seq_len_k, double softmax_scale, bool causal, bool return_lse) {
    const bool packed = cu_seqlens_q.has_value() && cu_seqlens_q->defined();
    TORCH_CHECK(packed == (cu_seqlens_k.has_value() && cu_seqlens_k->defined()),
                "mla_prefill: cu_seqlens_q and cu_seqlens_k come together");
    const int64_t lead = packed ? 1 : 2;
    const bool bf16 = query.scalar_type() == at::kBFloat16;
    TORCH_CHECK(query.scalar_type() == at::kHalf || bf16, "mla_prefill: float16 or bfloat16 inputs expected");
    // elements from one row to the next (dense sequences of one row: from one to the next)
    auto row_stride = [&](const at::Tensor &t) { return !packed && t.size(1) == 1 ? t.stride(0) : t.stride(lead - 1); };
    auto check = [&](const at::Tensor &t, const char *name, int64_t heads, int64_t width) {
        TORCH_CHECK(t.is_cuda() && t.device() == query.device(), name, " must be a CUDA tensor on the query's device");
        TORCH_CHECK(t.scalar_type() == query.scalar_type(), "mla_prefill: ", name, " must have the query's dtype");
        TORCH_CHECK(t.dim() == lead + (heads > 0 ? 2 : 1) && t.size(-1) == width && (heads <= 0 || t.size(-2) == heads),
                    "mla_prefill: ", name, " has the wrong shape");
        TORCH_CHECK(t.numel() == 0 || t.stride(-1) == 1, "mla_prefill: ", name, " must have a dense last dimension");
        TORCH_CHECK(packed || t.size(0) <= 1 || t.size(1) <= 1 || t.stride(0) == t.size(1) * t.stride(1),
                    "mla_prefill: ", name, "'s sequences must follow one another");
        const int64_t rows = packed ? t.size(0) : t.size(0) * t.size(1);
        TORCH_CHECK(t.numel() == 0 || (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                                       (rows <= 1 || row_stride(t) % 8 == 0) && (heads <= 1 || t.stride(lead) % 8 == 0)),
                    "mla_prefill: ", name, " must start and step in multiples of 16 bytes");
    };
    TORCH_CHECK(query.is_cuda() && query.dim() == lead + 2 && query.size(-2) >= 1,
                "mla_prefill: query must be a CUDA tensor [Tq, n_h, 192] (packed) or [B, Lq, n_h, 192]");
    const int64_t nh = query.size(-2);
    check(query, "query", nh, MLA_B200_HEAD_DIM + MLA_B200_HEAD_DIM_ROPE);
    check(k_nope, "k_nope", nh, MLA_B200_HEAD_DIM);
    check(v, "v", nh, MLA_B200_HEAD_DIM);
    check(k_rope, "k_rope", 0, MLA_B200_HEAD_DIM_ROPE);
    for (int64_t d = 0; d < lead; ++d)
        TORCH_CHECK(k_nope.size(d) == v.size(d) && k_nope.size(d) == k_rope.size(d) &&
                        (packed || d > 0 || k_nope.size(0) == query.size(0)),
                    "mla_prefill: k_nope, k_rope and v must have the same tokens");
    c10::cuda::CUDAGuard g(query.device());
    const int32_t *cu_q = nullptr, *cu_k = nullptr;
    int64_t b = query.size(0), tq = query.size(0), tk = k_nope.size(0);
    if (packed) {
        for (const at::Tensor *cu : {&*cu_seqlens_q, &*cu_seqlens_k}) {
            check_cuda(*cu, "cu_seqlens");
            TORCH_CHECK(cu->device() == query.device() && cu->scalar_type() == at::kInt && cu->dim() == 1 &&
                            cu->size(0) >= 1 && cu->size(0) == cu_seqlens_q->size(0),
                        "mla_prefill: cu_seqlens must be int32 [B + 1] on the query's device");
        }
        b = cu_seqlens_q->size(0) - 1;
        cu_q = cu_seqlens_q->data_ptr<int32_t>();
        cu_k = cu_seqlens_k->data_ptr<int32_t>();
        auto longest = [&](const at::Tensor &cu) {
            return b > 0 ? std::max<int64_t>((cu.slice(0, 1) - cu.slice(0, 0, b)).max().item<int64_t>(), 0) : 0;
        };
        if (max_seq_len_q < 0) max_seq_len_q = longest(*cu_seqlens_q);
        if (max_seq_len_k < 0) max_seq_len_k = longest(*cu_seqlens_k);
    } else {
        max_seq_len_q = query.size(1);
        max_seq_len_k = k_nope.size(1);
        tq = b * max_seq_len_q;
        tk = b * max_seq_len_k;
    }
    TORCH_CHECK(max_seq_len_q <= INT32_MAX && max_seq_len_k <= INT32_MAX && b <= INT32_MAX && nh <= INT32_MAX,
                "mla_prefill: sizes out of range");
    auto shape = query.sizes().vec();
    shape.back() = MLA_B200_HEAD_DIM;
    // (rows outside every sequence of a packed batch are left as they are allocated)
    at::Tensor out = fresh(shape, query.scalar_type(), query);
    shape.pop_back();
    if (!return_lse) shape[0] = 0;
    at::Tensor lse = fresh(shape, at::kFloat, query);
    const size_t ws = mla_b200_workspace_size_prefill((int)b, (int)nh, tq, (int)max_seq_len_q, (int)max_seq_len_k);
    at::Tensor w = fresh({(int64_t)std::max<size_t>(ws, 256)}, at::kByte, query);
    auto *fn = bf16 ? mla_b200_prefill_bf16 : mla_b200_prefill_f16;
    const int64_t d = lead - 1;
    check_status(fn(query.data_ptr(), row_stride(query), query.stride(d + 1), k_nope.data_ptr(), row_stride(k_nope),
                    k_nope.stride(d + 1), k_rope.data_ptr(), row_stride(k_rope), v.data_ptr(), row_stride(v),
                    v.stride(d + 1), cu_q, cu_k, (int)b, (int)nh, tq, tk, (int)max_seq_len_q, (int)max_seq_len_k,
                    causal ? 1 : 0, (float)softmax_scale, out.data_ptr(), return_lse ? lse.data_ptr<float>() : nullptr,
                    w.data_ptr(), ws, stream_ptr()),
                 "mla_prefill");
    return {out, lse};
}

// Pages and slots for a step's new tokens (no reference counterpart); block_table is
// written in place.  Returns (slots int64 [num_tokens], positions int32
// [num_tokens], cu_new int32 [B + 1], new seq_lens int32 [B], new free_head int32 [1]).
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> mla_build_slots(
    const at::Tensor &seq_lens, const at::Tensor &new_lens, at::Tensor block_table, const at::Tensor &free_pages,
    int64_t page_size, int64_t num_tokens, const c10::optional<at::Tensor> &free_head) {
    check_cuda(seq_lens, "seq_lens");
    check_cuda(new_lens, "new_lens");
    check_cuda(free_pages, "free_pages");
    TORCH_CHECK(block_table.is_cuda(), "block_table must be a CUDA tensor");
    const int64_t b = seq_lens.size(0);
    TORCH_CHECK(seq_lens.dim() == 1 && new_lens.dim() == 1 && new_lens.size(0) == b &&
                    seq_lens.scalar_type() == at::kInt && new_lens.scalar_type() == at::kInt,
                "mla_build_slots: seq_lens and new_lens must be int32 [B]");
    TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == b &&
                    (block_table.size(1) <= 1 || block_table.stride(1) == 1) &&
                    (b <= 1 || block_table.stride(0) >= block_table.size(1)),
                "mla_build_slots: block_table must be int32 [B, max_blocks] with dense rows");
    TORCH_CHECK(free_pages.scalar_type() == at::kInt && free_pages.dim() == 1,
                "mla_build_slots: free_pages must be int32 [F]");
    TORCH_CHECK(page_size >= 1 && page_size <= INT32_MAX && num_tokens >= 0 && num_tokens <= INT32_MAX &&
                    free_pages.size(0) <= INT32_MAX && block_table.size(1) <= INT32_MAX && b <= INT32_MAX,
                "mla_build_slots: page_size or num_tokens out of range");
    TORCH_CHECK(seq_lens.device() == new_lens.device() && seq_lens.device() == block_table.device() &&
                    seq_lens.device() == free_pages.device(),
                "mla_build_slots: all tensors on one device");
    const int32_t *head = nullptr;
    if (free_head.has_value() && free_head->defined()) {
        check_cuda(*free_head, "free_head");
        TORCH_CHECK(free_head->scalar_type() == at::kInt && free_head->numel() == 1 &&
                        free_head->device() == seq_lens.device(),
                    "mla_build_slots: free_head must be one int32 on the same device");
        head = free_head->data_ptr<int32_t>();
    }
    c10::cuda::CUDAGuard g(seq_lens.device());
    // A caller keeps the lengths and the head from step to step.  In one allocation with the
    // tokens' 12 bytes each they would keep those too, so that is for small steps alone (256
    // tokens: 8.8 us a call, 9.5 with two allocations; 381 000 tokens: 10.2 either way).
    const bool together = num_tokens <= 4096;
    const int64_t token_bytes = Carve::room(num_tokens, 8) + Carve::room(num_tokens, 4);
    const int64_t request_bytes = Carve::room(b + 1, 4) + Carve::room(b, 4) + 16;
    Carve of_tokens(token_bytes + (together ? request_bytes : 0), seq_lens);
    at::Tensor slots = of_tokens.take(num_tokens, at::kLong), positions = of_tokens.take(num_tokens, at::kInt);
    Carve of_requests = together ? of_tokens : Carve(request_bytes, seq_lens);
    at::Tensor cu_new = of_requests.take(b + 1, at::kInt), lens = of_requests.take(b, at::kInt);
    at::Tensor new_head = of_requests.take(1, at::kInt);
    check_status(mla_b200_build_slots(seq_lens.data_ptr<int32_t>(), new_lens.data_ptr<int32_t>(),
                                      block_table.data_ptr<int32_t>(),
                                      b > 1 ? block_table.stride(0) : block_table.size(1), (int)block_table.size(1),
                                      free_pages.data_ptr<int32_t>(), (int)free_pages.size(0), head, (int)b,
                                      (int)page_size, (int)num_tokens, slots.data_ptr<int64_t>(),
                                      positions.data_ptr<int32_t>(), cu_new.data_ptr<int32_t>(),
                                      lens.data_ptr<int32_t>(), new_head.data_ptr<int32_t>(), stream_ptr()),
                 "mla_build_slots");
    return {slots, positions, cu_new, lens, new_head};
}

// Latent rows into the cache (no reference counterpart); cache (and kv_scales) are
// written in place.
void mla_cache_write(const at::Tensor &latent, const at::Tensor &slots, at::Tensor cache,
                     const c10::optional<at::Tensor> &norm_weight, double eps,
                     const c10::optional<at::Tensor> &positions, const c10::optional<at::Tensor> &cos_sin,
                     bool interleaved, const c10::optional<at::Tensor> &kv_scales) {
    TORCH_CHECK(latent.is_cuda(), "latent must be a CUDA tensor");
    check_cuda(slots, "slots");
    check_cuda(cache, "cache");
    auto dtype_of = [](at::ScalarType t) {
        return t == at::kHalf ? (int)MLA_B200_DTYPE_F16
               : t == at::kBFloat16 ? (int)MLA_B200_DTYPE_BF16
               : t == at::kFloat ? (int)MLA_B200_DTYPE_F32
               : t == at::kFloat8_e4m3fn ? (int)MLA_B200_DTYPE_E4M3 : -1;
    };
    const int in = dtype_of(latent.scalar_type()), to = dtype_of(cache.scalar_type());
    TORCH_CHECK(in >= 0 && in != MLA_B200_DTYPE_E4M3,
                "mla_cache_write: float16, bfloat16 or float32 latent rows expected");
    TORCH_CHECK(to >= 0 && to != MLA_B200_DTYPE_F32,
                "mla_cache_write: a float16, bfloat16 or float8_e4m3fn cache expected");
    const int64_t t = latent.dim() == 2 ? latent.size(0) : -1;
    TORCH_CHECK(t >= 0 && t <= INT32_MAX && latent.size(1) == MLA_B200_HEAD_DIM_K && latent.stride(1) == 1,
                "mla_cache_write: latent must be [T, 576] with dense rows");
    TORCH_CHECK(slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.size(0) == t,
                "mla_cache_write: slots must be int64 [T]");
    TORCH_CHECK((cache.dim() == 2 || cache.dim() == 3) && cache.size(-1) == MLA_B200_HEAD_DIM_K,
                "mla_cache_write: cache must be [rows, 576] or [num_pages, page_size, 576]");
    TORCH_CHECK(latent.device() == slots.device() && latent.device() == cache.device(),
                "mla_cache_write: all tensors on one device");
    const int64_t rows = cache.numel() / MLA_B200_HEAD_DIM_K;
    const void *w = nullptr;
    if (norm_weight.has_value() && norm_weight->defined()) {
        check_cuda(*norm_weight, "norm_weight");
        TORCH_CHECK(norm_weight->scalar_type() == latent.scalar_type() && norm_weight->device() == latent.device() &&
                        norm_weight->dim() == 1 && norm_weight->size(0) == MLA_B200_HEAD_DIM_V,
                    "mla_cache_write: norm_weight must be [512] in the latent rows' dtype");
        w = norm_weight->data_ptr();
    }
    const int32_t *pos = nullptr;
    const float *cs = nullptr;
    int max_pos = 0;
    const bool has_pos = positions.has_value() && positions->defined();
    TORCH_CHECK(has_pos == (cos_sin.has_value() && cos_sin->defined()),
                "mla_cache_write: positions and cos_sin come together");
    if (has_pos) {
        check_cuda(*positions, "positions");
        check_cuda(*cos_sin, "cos_sin");
        TORCH_CHECK(positions->scalar_type() == at::kInt && positions->dim() == 1 && positions->size(0) == t &&
                        positions->device() == latent.device(),
                    "mla_cache_write: positions must be int32 [T]");
        TORCH_CHECK(cos_sin->scalar_type() == at::kFloat && cos_sin->dim() == 2 && cos_sin->size(0) <= INT32_MAX &&
                        cos_sin->size(1) == MLA_B200_HEAD_DIM_ROPE && cos_sin->device() == latent.device(),
                    "mla_cache_write: cos_sin must be float32 [max_positions, 64]");
        pos = positions->data_ptr<int32_t>();
        cs = cos_sin->data_ptr<float>();
        max_pos = (int)cos_sin->size(0);
    }
    float *scales = nullptr;
    const bool has_scales = kv_scales.has_value() && kv_scales->defined();
    TORCH_CHECK(has_scales == (to == MLA_B200_DTYPE_E4M3),
                "mla_cache_write: kv_scales goes with a float8_e4m3fn cache, and only with one");
    if (has_scales) {
        check_cuda(*kv_scales, "kv_scales");
        TORCH_CHECK(kv_scales->scalar_type() == at::kFloat && kv_scales->numel() == rows &&
                        kv_scales->device() == latent.device(),
                    "mla_cache_write: kv_scales must be float32, one per cache row");
        scales = kv_scales->data_ptr<float>();
    }
    c10::cuda::CUDAGuard g(latent.device());
    check_status(mla_b200_cache_write(latent.data_ptr(), in, t > 1 ? latent.stride(0) : MLA_B200_HEAD_DIM_K,
                                      slots.data_ptr<int64_t>(), (int)t, w, (float)eps, pos, cs, max_pos,
                                      interleaved ? 1 : 0, cache.data_ptr(), to, rows, scales, stream_ptr()),
                 "mla_cache_write");
}

// LSE merge of partials: part_o [P, rows, 512] fp32, part_lse [P, rows] fp32.
std::vector<at::Tensor> mla_combine(const at::Tensor &part_o, const at::Tensor &part_lse,
                                    bool out_fp32) {
    check_cuda(part_o, "part_o");
    check_cuda(part_lse, "part_lse");
    TORCH_CHECK(part_o.scalar_type() == at::kFloat && part_lse.scalar_type() == at::kFloat,
                "mla_combine: float32 partials expected");
    TORCH_CHECK(part_o.dim() == 3 && part_o.size(2) == MLA_B200_HEAD_DIM_V && part_lse.dim() == 2 &&
                    part_lse.size(0) == part_o.size(0) && part_lse.size(1) == part_o.size(1),
                "mla_combine: expected part_o [P, rows, 512] and part_lse [P, rows]");
    c10::cuda::CUDAGuard g(part_o.device());
    const int64_t p = part_o.size(0), rows = part_o.size(1);
    at::Tensor out = at::empty({rows, MLA_B200_HEAD_DIM_V},
                               part_o.options().dtype(out_fp32 ? at::kFloat : at::kHalf));
    at::Tensor lse = at::empty({rows}, part_o.options());
    check_status(mla_b200_combine_f32(part_o.data_ptr<float>(), part_lse.data_ptr<float>(), (int)p,
                                      rows, out.data_ptr(),
                                      out_fp32 ? MLA_B200_OUT_F32 : MLA_B200_OUT_F16,
                                      lse.data_ptr<float>(), stream_ptr()),
                 "mla_combine");
    return {out, lse};
}

int64_t mla_get_device_error() {
    int code = 0;
    const int st = mla_b200_get_device_error(&code, stream_ptr());
    TORCH_CHECK(st == MLA_B200_OK || st == MLA_B200_ERR_DEVICE_TIMEOUT,
                "mla_get_device_error failed: ", mla_b200_status_string(st));
    return code;
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("mla_decode_naive", &mla_decode_naive, "fp32 naive decode, reference semantics",
          py::arg("query"), py::arg("cache"));
    m.def("mla_decode_fused", &mla_decode_fused, "fp32 fused decode, reference semantics",
          py::arg("query"), py::arg("cache"));
    m.def("mla_decode_split", &mla_decode_split, "split-KV decode, reference semantics",
          py::arg("query"), py::arg("cache"), py::arg("num_splits") = -1);
    m.def("mla_decode_batched", &mla_decode_batched, "batched / varlen decode (fp16, bf16, fp8 cache)",
          py::arg("query"), py::arg("cache"), py::arg("cu_seqlens") = py::none(),
          py::arg("max_seq_len") = -1, py::arg("softmax_scale") = 0.07216878364870322,
          py::arg("num_splits") = -1, py::arg("return_lse") = false, py::arg("out_fp32") = false,
          py::arg("kv_scale") = 1.0);
    m.def("mla_decode_mtp", &mla_decode_mtp, "multi-token (draft) decode sharing each cache tile",
          py::arg("query"), py::arg("cache"), py::arg("cu_seqlens") = py::none(),
          py::arg("max_seq_len") = -1, py::arg("softmax_scale") = 0.07216878364870322,
          py::arg("num_splits") = -1, py::arg("return_lse") = false, py::arg("out_fp32") = false);
    m.def("mla_decode_paged", &mla_decode_paged, "decode over a paged latent cache",
          py::arg("query"), py::arg("kv_pages"), py::arg("block_table"), py::arg("seq_lens"),
          py::arg("max_seq_len") = -1, py::arg("softmax_scale") = 0.07216878364870322,
          py::arg("num_splits") = -1, py::arg("return_lse") = false, py::arg("out_fp32") = false);
    m.def("mla_decode_tree", &mla_decode_tree, "draft-tree decode over a paged latent cache",
          py::arg("query"), py::arg("kv_pages"), py::arg("block_table"), py::arg("seq_lens"),
          py::arg("tree_mask") = py::none(), py::arg("max_seq_len") = -1,
          py::arg("softmax_scale") = 0.07216878364870322, py::arg("num_splits") = -1,
          py::arg("return_lse") = false, py::arg("out_fp32") = false);
    m.def("mla_prefill", &mla_prefill, "attention over prompts in expanded form", py::arg("query"),
          py::arg("k_nope"), py::arg("k_rope"), py::arg("v"), py::arg("cu_seqlens_q") = py::none(),
          py::arg("cu_seqlens_k") = py::none(), py::arg("max_seq_len_q") = -1, py::arg("max_seq_len_k") = -1,
          py::arg("softmax_scale") = 0.07216878364870322, py::arg("causal") = true, py::arg("return_lse") = false);
    m.def("mla_build_slots", &mla_build_slots, "pages and slots for a step's new tokens", py::arg("seq_lens"),
          py::arg("new_lens"), py::arg("block_table"), py::arg("free_pages"), py::arg("page_size"),
          py::arg("num_tokens"), py::arg("free_head") = py::none());
    m.def("mla_cache_write", &mla_cache_write, "latent rows into the cache", py::arg("latent"), py::arg("slots"),
          py::arg("cache"), py::arg("norm_weight") = py::none(), py::arg("eps") = 1e-6,
          py::arg("positions") = py::none(), py::arg("cos_sin") = py::none(), py::arg("interleaved") = true,
          py::arg("kv_scales") = py::none());
    m.def("mla_combine", &mla_combine, "log-sum-exp merge of partial decodes", py::arg("part_o"),
          py::arg("part_lse"), py::arg("out_fp32") = false);
    m.def("mla_get_device_error", &mla_get_device_error,
          "read and clear the kernels' device error word");
    m.attr("NUM_HEADS") = MLA_B200_NUM_HEADS;
    m.attr("HEAD_DIM") = MLA_B200_HEAD_DIM;
    m.attr("HEAD_DIM_C") = MLA_B200_HEAD_DIM_C;
    m.attr("HEAD_DIM_ROPE") = MLA_B200_HEAD_DIM_ROPE;
    m.attr("HEAD_DIM_K") = MLA_B200_HEAD_DIM_K;
    m.attr("HEAD_DIM_V") = MLA_B200_HEAD_DIM_V;
}
