// Entry points of the linear and the gated layer (head_layer_impl.h).
#include "head_layer.h"

namespace collie {
namespace {

int check_layer(const char* who, int64_t m, int32_t n_in, int32_t n_out, int64_t x_ld, int32_t act) {
  COLLIE_REQUIRE(m >= 0 && m < (int64_t{1} << 31), "%s: bad number of rows", who);
  COLLIE_REQUIRE(n_in >= 1 && n_out >= 1 && n_in <= (1 << 19) && n_out <= (1 << 19),
                 "%s: widths must be in [1, 2^19]", who);
  COLLIE_REQUIRE(m <= 1 || x_ld >= n_in, "%s: rows of x overlap", who);
  COLLIE_REQUIRE(act >= COLLIE_ACT_IDENTITY && act <= COLLIE_ACT_GELU, "%s: unknown activation %d",
                 who, act);
  return 0;
}

}  // namespace
}  // namespace collie

using namespace collie;

extern "C" size_t collie_layer_forward_workspace_bytes(const void* x, int64_t x_ld, int32_t dtype,
                                                       int64_t m, int32_t n_in, const void* weight,
                                                       const void* up_weight, int32_t n_out) {
  if (m < 1 || n_in < 1 || n_out < 1) return 256;
  size_t bytes = 0;
  with_type(dtype, "layer_forward", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    bytes = HeadLayer<T>::forward_bytes(x, x_ld, m, n_in, weight, up_weight, n_out);
    return 0;
  });
  return bytes;
}

extern "C" size_t collie_layer_backward_workspace_bytes(const void* dy, int64_t dy_ld, const void* x,
                                                        int64_t x_ld, int32_t dtype, int64_t m,
                                                        int32_t n_in, const void* weight,
                                                        const void* up_weight, int32_t n_out,
                                                        int32_t act) {
  if (m < 1 || n_in < 1 || n_out < 1) return 256;
  size_t bytes = 0;
  with_type(dtype, "layer_backward", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    bytes = HeadLayer<T>::backward_bytes(dy, dy_ld, x, x_ld, m, n_in, weight, up_weight, n_out, act);
    return 0;
  });
  return bytes;
}

extern "C" int collie_layer_plan(int32_t dtype, int32_t product, int32_t gated, int64_t m, int32_t n_in,
                                 int32_t n_out, int64_t* plan) {
  if (check_layer("layer_plan", m, n_in, n_out, n_in, COLLIE_ACT_IDENTITY)) return -1;
  COLLIE_REQUIRE(m >= 1 && plan, "layer_plan: no rows or no room for the plan");
  COLLIE_REQUIRE(product >= COLLIE_PRODUCT_FORWARD && product <= COLLIE_PRODUCT_DW,
                 "layer_plan: unknown product %d", product);
  return with_type(dtype, "layer_plan", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    int64_t out[5];
    HeadLayer<T>::plan(static_cast<Product>(product), m, n_in, n_out, gated != 0, out);
    memcpy(plan, out, sizeof(out));
    return 0;
  });
}

extern "C" int collie_linear_forward(const void* x, int64_t x_ld, int32_t dtype, int64_t m,
                                     int32_t n_in, const void* weight, const void* bias,
                                     int32_t n_out, int32_t act, const void* residual,
                                     int64_t res_ld, void* keep, void* y, void* workspace,
                                     size_t workspace_bytes, collie_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (check_layer("linear_forward", m, n_in, n_out, x_ld, act)) return -1;
  COLLIE_REQUIRE(!residual || m <= 1 || res_ld >= n_out, "linear_forward: rows of residual overlap");
  if (m == 0) return 0;
  COLLIE_REQUIRE(x && weight && y, "linear_forward: NULL pointer");
  const size_t need =
      collie_layer_forward_workspace_bytes(x, x_ld, dtype, m, n_in, weight, nullptr, n_out);
  COLLIE_REQUIRE(workspace && workspace_bytes >= need, "workspace too small: need %zu bytes, got %zu",
                 need, workspace_bytes);
  return with_type(dtype, "linear_forward", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    return HeadLayer<T>::forward(x, x_ld, weight, nullptr, bias, nullptr, residual, res_ld, m, n_in,
                            n_out, act, keep, nullptr, y, workspace, stream);
  });
}

extern "C" int collie_gated_forward(const void* x, int64_t x_ld, int32_t dtype, int64_t m,
                                    int32_t n_in, const void* gate_weight, const void* up_weight,
                                    const void* gate_bias, const void* up_bias, int32_t n_out,
                                    int32_t act, void* keep_gate, void* keep_up, void* y,
                                    void* workspace, size_t workspace_bytes,
                                    collie_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (check_layer("gated_forward", m, n_in, n_out, x_ld, act)) return -1;
  COLLIE_REQUIRE((gate_bias == nullptr) == (up_bias == nullptr),
                 "gated_forward: both biases or none");
  COLLIE_REQUIRE((keep_gate == nullptr) == (keep_up == nullptr),
                 "gated_forward: keep_gate and keep_up belong together");
  if (m == 0) return 0;
  COLLIE_REQUIRE(x && gate_weight && up_weight && y, "gated_forward: NULL pointer");
  const size_t need =
      collie_layer_forward_workspace_bytes(x, x_ld, dtype, m, n_in, gate_weight, up_weight, n_out);
  COLLIE_REQUIRE(workspace && workspace_bytes >= need, "workspace too small: need %zu bytes, got %zu",
                 need, workspace_bytes);
  return with_type(dtype, "gated_forward", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    return HeadLayer<T>::forward(x, x_ld, gate_weight, up_weight, gate_bias, up_bias, nullptr, 0, m, n_in,
                            n_out, act, keep_gate, keep_up, y, workspace, stream);
  });
}

extern "C" int collie_linear_backward(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld,
                                      int32_t dtype, int64_t m, int32_t n_in, const void* weight,
                                      int32_t n_out, int32_t act, const void* kept_z, void* dx,
                                      void* dweight, void* dbias, void* workspace,
                                      size_t workspace_bytes, collie_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (check_layer("linear_backward", m, n_in, n_out, x_ld, act)) return -1;
  COLLIE_REQUIRE(m <= 1 || dy_ld >= n_out, "linear_backward: rows of dy overlap");
  COLLIE_REQUIRE(m >= 1, "linear_backward: no rows");
  COLLIE_REQUIRE(dy && x && weight, "linear_backward: NULL pointer");
  COLLIE_REQUIRE((act == COLLIE_ACT_IDENTITY) == (kept_z == nullptr),
                 "linear_backward: kept_z is what the forward pass kept (NULL for the identity)");
  const size_t need = collie_layer_backward_workspace_bytes(dy, dy_ld, x, x_ld, dtype, m, n_in,
                                                            weight, nullptr, n_out, act);
  COLLIE_REQUIRE(workspace && workspace_bytes >= need, "workspace too small: need %zu bytes, got %zu",
                 need, workspace_bytes);
  return with_type(dtype, "linear_backward", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    return HeadLayer<T>::backward(dy, dy_ld, x, x_ld, weight, nullptr, kept_z, nullptr, m, n_in, n_out,
                             act, dx, dweight, nullptr, dbias, nullptr, workspace, stream);
  });
}

extern "C" int collie_gated_backward(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld,
                                     int32_t dtype, int64_t m, int32_t n_in, const void* gate_weight,
                                     const void* up_weight, int32_t n_out, int32_t act,
                                     const void* kept_gate, const void* kept_up, void* dx,
                                     void* dgate_weight, void* dup_weight, void* dgate_bias,
                                     void* dup_bias, void* workspace, size_t workspace_bytes,
                                     collie_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (check_layer("gated_backward", m, n_in, n_out, x_ld, act)) return -1;
  COLLIE_REQUIRE(m <= 1 || dy_ld >= n_out, "gated_backward: rows of dy overlap");
  COLLIE_REQUIRE(m >= 1, "gated_backward: no rows");
  COLLIE_REQUIRE(dy && x && gate_weight && up_weight && kept_gate && kept_up,
                 "gated_backward: NULL pointer");
  const size_t need = collie_layer_backward_workspace_bytes(
      dy, dy_ld, x, x_ld, dtype, m, n_in, gate_weight, up_weight, n_out, act);
  COLLIE_REQUIRE(workspace && workspace_bytes >= need, "workspace too small: need %zu bytes, got %zu",
                 need, workspace_bytes);
  return with_type(dtype, "gated_backward", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    return HeadLayer<T>::backward(dy, dy_ld, x, x_ld, gate_weight, up_weight, kept_gate, kept_up, m, n_in,
                             n_out, act, dx, dgate_weight, dup_weight, dgate_bias, dup_bias,
                             workspace, stream);
  });
}
