// Python module `pos_encoding_ops`: same name, function and argument order as
// vLLM v0.1.0's csrc/pos_encoding.cpp:3-15, so
// vllm/model_executor/layers/attention.py:200-206 calls it unchanged.
#include "torch_shim.h"

namespace {

void rotary_embedding_neox(torch::Tensor& positions,      // [num_tokens]
                           torch::Tensor& query,          // [num_tokens, num_heads * head_size]
                           torch::Tensor& key,            // [num_tokens, num_heads * head_size]
                           int head_size,
                           torch::Tensor& cos_sin_cache)  // [max_position, rot_dim]
{
  using namespace pa_shim;
  const char* what = "rotary_embedding_neox";
  TORCH_CHECK(positions.is_cuda() && query.is_cuda() && key.is_cuda() && cos_sin_cache.is_cuda(), what,
              ": all tensors must be on the GPU");
  const int dtype = dtype_code(query, what);
  TORCH_CHECK(key.scalar_type() == query.scalar_type() && cos_sin_cache.scalar_type() == query.scalar_type(), what,
              ": query, key and cos_sin_cache must share one data type");
  TORCH_CHECK(positions.scalar_type() == at::ScalarType::Long && positions.is_contiguous(), what,
              ": positions must be a contiguous int64 tensor");
  TORCH_CHECK(query.dim() == 2 && key.dim() == 2 && query.sizes() == key.sizes(), what,
              ": query and key must be [num_tokens, num_heads * head_size]");
  TORCH_CHECK(query.size(0) == 0 || (query.stride(1) == 1 && key.stride(1) == 1), what,
              ": query and key rows must be dense");
  TORCH_CHECK(head_size > 0 && query.size(1) % head_size == 0, what, ": hidden size is not a multiple of head_size");
  TORCH_CHECK(cos_sin_cache.dim() == 2 && cos_sin_cache.is_contiguous(), what,
              ": cos_sin_cache must be a contiguous [max_position, rot_dim] tensor");
  const int num_tokens = query.size(0);
  TORCH_CHECK(positions.numel() >= num_tokens, what, ": positions is shorter than the number of tokens");
  // the reference requires equal row strides (pos_encoding_kernels.cu:62)
  TORCH_CHECK(num_tokens == 0 || query.stride(0) == key.stride(0), what, ": query and key row strides differ");
  PA_DEVICE_GUARD(query);
  check_status(pa_rotary_embedding_neox(positions.data_ptr<int64_t>(), query.data_ptr(), key.data_ptr(),
                                        cos_sin_cache.data_ptr(), num_tokens,
                                        static_cast<int>(query.size(1) / head_size), head_size,
                                        static_cast<int>(cos_sin_cache.size(1)),
                                        num_tokens > 0 ? query.stride(0) : 0, num_tokens > 0 ? key.stride(0) : 0,
                                        dtype, current_stream(query)),
               what);
}

// Not part of the reference's module: both pair layouts, numbers of query and key heads of their own,
// a float32 table beside 16-bit rows, one rounding at the end.  A negative position leaves its row as
// it is (padding); one past the table fills what it would rotate with NaN.
struct RotaryCall {
  int num_tokens, num_heads, num_kv_heads, rot_dim, dtype, table_dtype;
  int64_t max_position, query_stride, key_stride;
};

RotaryCall check_rotary(const char* what, const torch::Tensor& positions, const torch::Tensor& query,
                        const torch::Tensor& key, int64_t head_size, const torch::Tensor& cos_sin_cache) {
  using namespace pa_shim;
  TORCH_CHECK(positions.is_cuda() && query.is_cuda() && key.is_cuda() && cos_sin_cache.is_cuda(), what,
              ": all tensors must be on the GPU");
  check_one_device(what, query, {&positions, &key, &cos_sin_cache});
  RotaryCall c;
  c.dtype = dtype_code(query, what);
  TORCH_CHECK(key.scalar_type() == query.scalar_type(), what, ": query and key must share one data type");
  TORCH_CHECK(cos_sin_cache.scalar_type() == at::ScalarType::Float || cos_sin_cache.scalar_type() == query.scalar_type(),
              what, ": cos_sin_cache must be float32 or of query's data type");
  c.table_dtype = dtype_code(cos_sin_cache, what);
  TORCH_CHECK(positions.scalar_type() == at::ScalarType::Long && positions.is_contiguous(), what,
              ": positions must be a contiguous int64 tensor");
  TORCH_CHECK(query.dim() == 2 && key.dim() == 2 && query.size(0) == key.size(0), what,
              ": query must be [num_tokens, num_heads * head_size] and key [num_tokens, num_kv_heads * head_size]");
  TORCH_CHECK((query.numel() == 0 || query.size(1) == 1 || query.stride(1) == 1) &&
                  (key.numel() == 0 || key.size(1) == 1 || key.stride(1) == 1),
              what, ": query and key rows must be dense");
  TORCH_CHECK(head_size > 0 && head_size <= (1 << 20) && query.size(1) % head_size == 0 && key.size(1) % head_size == 0, what,
              ": the rows are no multiple of head_size");
  TORCH_CHECK(cos_sin_cache.dim() == 2 && cos_sin_cache.is_contiguous() && cos_sin_cache.size(1) <= head_size, what,
              ": cos_sin_cache must be a contiguous [max_position, rot_dim] tensor, rot_dim at most head_size");
  TORCH_CHECK(query.size(0) <= INT32_MAX && query.size(1) <= INT32_MAX && key.size(1) <= INT32_MAX, what, ": too many rows");
  TORCH_CHECK(positions.numel() >= query.size(0), what, ": positions is shorter than the number of tokens");
  c.num_tokens = query.size(0);
  c.num_heads = query.size(1) / head_size;
  c.num_kv_heads = key.size(1) / head_size;
  c.rot_dim = cos_sin_cache.size(1);
  c.max_position = cos_sin_cache.size(0);
  c.query_stride = query.stride(0);
  c.key_stride = key.stride(0);
  return c;
}

void rotary_embedding(const torch::Tensor& positions,      // [num_tokens]
                      const torch::Tensor& query,          // [num_tokens, num_heads * head_size]
                      const torch::Tensor& key,            // [num_tokens, num_kv_heads * head_size]
                      int64_t head_size,
                      const torch::Tensor& cos_sin_cache,  // [max_position, rot_dim]
                      bool interleaved) {
  using namespace pa_shim;
  const char* what = "rotary_embedding";
  const RotaryCall c = check_rotary(what, positions, query, key, head_size, cos_sin_cache);
  PA_DEVICE_GUARD(query);
  check_status(pa_rotary_embedding(positions.data_ptr<int64_t>(), query.data_ptr(), key.data_ptr(),
                                   cos_sin_cache.data_ptr(), c.num_tokens, c.num_heads, c.num_kv_heads,
                                   static_cast<int>(head_size), c.rot_dim, c.max_position, c.query_stride, c.key_stride,
                                   interleaved, c.dtype, c.table_dtype, current_stream(query)),
               what);
}

void qk_norm_rotary_embedding(const torch::Tensor& positions, const torch::Tensor& query, const torch::Tensor& key,
                              int64_t head_size,
                              const torch::Tensor& query_weight,  // [head_size]
                              const torch::Tensor& key_weight,    // [head_size]
                              double epsilon, const torch::Tensor& cos_sin_cache, bool interleaved) {
  using namespace pa_shim;
  const char* what = "qk_norm_rotary_embedding";
  const RotaryCall c = check_rotary(what, positions, query, key, head_size, cos_sin_cache);
  TORCH_CHECK(query_weight.is_cuda() && key_weight.is_cuda(), what, ": all tensors must be on the GPU");
  check_one_device(what, query, {&query_weight, &key_weight});
  TORCH_CHECK(query_weight.scalar_type() == query.scalar_type() && key_weight.scalar_type() == query.scalar_type(), what,
              ": the weights must be of query's data type");
  TORCH_CHECK(query_weight.is_contiguous() && key_weight.is_contiguous() && query_weight.numel() == head_size &&
                  key_weight.numel() == head_size,
              what, ": the weights must be [head_size]");
  TORCH_CHECK(epsilon >= 0, what, ": epsilon must not be negative");
  PA_DEVICE_GUARD(query);
  check_status(pa_qk_norm_rotary_embedding(
                   positions.data_ptr<int64_t>(), query.data_ptr(), key.data_ptr(), query_weight.data_ptr(),
                   key_weight.data_ptr(), static_cast<float>(epsilon), cos_sin_cache.data_ptr(), c.num_tokens, c.num_heads,
                   c.num_kv_heads, static_cast<int>(head_size), c.rot_dim, c.max_position, c.query_stride, c.key_stride,
                   interleaved, c.dtype, c.table_dtype, current_stream(query)),
               what);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("rotary_embedding_neox", &rotary_embedding_neox,
        "Apply GPT-NeoX style rotary embedding to query and key, in place");
  m.def("rotary_embedding", &rotary_embedding,
        "Rotate the first rot_dim elements of every query and key head, in place: half or interleaved pairs, "
        "cos_sin_cache float32 or of query's type");
  m.def("qk_norm_rotary_embedding", &qk_norm_rotary_embedding,
        "RMS norm of every query and key head, then rotary_embedding, in one pass and in place");
}
