// The weight gradient's products of the linear layers: dW = dz^T x with x in its own type or in 8 bits, dz given, or dy and
// the forward pass' signs (the gate is applied on the way into LDS), and the bias gradient from the same pass over dz.
#define SG2IM_GEMM_TU 1
#include "linear.h"

namespace sg2im {
namespace lin {

template <typename T, int BMODE>
static int run_as(Product& p, const Plan& q, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (p.gate) return run<T, RM, BMODE, true, true>(p, q, workspace, workspace_bytes, stream);
  if (p.sum) return run<T, RM, BMODE, false, true>(p, q, workspace, workspace_bytes, stream);
  return run<T, RM, BMODE, false, false>(p, q, workspace, workspace_bytes, stream);
}

int run_weight(Product& p, int dtype, bool codes, const Plan& q, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (dtype == 0) return codes ? run_as<float, RM8>(p, q, workspace, workspace_bytes, stream) : run_as<float, RM>(p, q, workspace, workspace_bytes, stream);
  return codes ? run_as<bf16_s, RM8>(p, q, workspace, workspace_bytes, stream) : run_as<bf16_s, RM>(p, q, workspace, workspace_bytes, stream);
}

}  // namespace lin
}  // namespace sg2im
