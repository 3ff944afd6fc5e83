// The linear and the gated layer for one element type (w2 = NULL: linear).  Every type has a source
// file of its own, so that they are compiled side by side.
#pragma once

#include "head_gemm.h"

namespace collie {

enum Product { kForward = COLLIE_PRODUCT_FORWARD, kDx = COLLIE_PRODUCT_DX, kDw = COLLIE_PRODUCT_DW };

template <typename T>
struct HeadLayer {
  static void plan(Product product, int64_t m, int64_t n_in, int64_t n_out, bool pair,
                   int64_t (&out)[5]);
  static size_t forward_bytes(const void* x, int64_t x_ld, int64_t m, int64_t n_in, const void* w,
                              const void* w2, int64_t n_out);
  static size_t backward_bytes(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, int64_t m,
                               int64_t n_in, const void* w, const void* w2, int64_t n_out, int act);
  static int forward(const void* x, int64_t x_ld, const void* w, const void* w2, const void* bias,
                     const void* bias2, const void* residual, int64_t res_ld, int64_t m, int64_t n_in,
                     int64_t n_out, int act, void* keep, void* keep2, void* y, void* workspace,
                     hipStream_t stream);
  static int backward(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, const void* w,
                      const void* w2, const void* z, const void* u, int64_t m, int64_t n_in,
                      int64_t n_out, int act, void* dx, void* dw, void* dw2, void* db, void* db2,
                      void* workspace, hipStream_t stream);
};
extern template struct HeadLayer<float>;
extern template struct HeadLayer<bf16_t>;
extern template struct HeadLayer<f16_t>;

}  // namespace collie
