// =================================================================================================
// Xlayer<T>: host logic of the products of a network's layers - GemmEpilogue, GemmActivationGradient, ActivationGradient,
// GemmGrouped and GemmGroupedGradient (include/clblast_hip.h). All matrices are row-major; the routines check the
// arguments, read the row-major problem as the column-major one of the device layer (C^T = op(B)^T op(A)^T) and launch;
// the device layer copies an operand that cannot be fetched in dwords into the call's scratch memory.
// T is float, half or bfloat16. The reference has no such routines.
// =================================================================================================
#ifndef CLBLAST_HIP_ROUTINES_XLAYER_HPP_
#define CLBLAST_HIP_ROUTINES_XLAYER_HPP_

#include "routines/routine_common.hpp"
#include "routines/xgemm.hpp"

namespace clblast {
// =================================================================================================

// A caller's row-major matrix: its buffer, the first element, the distance of its rows
struct LayerMatrix {
  const void* pointer;
  size_t offset, ld;
};
// A caller's vectors: one per group, `stride` apart
struct LayerVector {
  const void* pointer;
  size_t offset, stride;
};
// The rows of the groups: group_count + 1 64-bit values on the device
struct LayerGroups {
  size_t count;
  const void* offsets;
  size_t offset;
};

template <typename T>
class Xlayer : public GemmRoutineBase {
 public:
  Xlayer(hipStream_t* queue, hipEvent_t* event);

  void DoGemmEpilogue(const Transpose a_transpose, const Transpose b_transpose, const size_t m, const size_t n, const size_t k,
                      const float alpha, const LayerMatrix& a, const LayerMatrix& b, const LayerVector& bias,
                      const Activation activation, const LayerMatrix& pre, const float beta, const LayerMatrix& residual,
                      const LayerMatrix& c);
  void DoGemmActivationGradient(const Transpose a_transpose, const Transpose b_transpose, const size_t m, const size_t n,
                                const size_t k, const float alpha, const LayerMatrix& a, const LayerMatrix& b,
                                const Activation activation, const LayerMatrix& pre, const LayerMatrix& c,
                                const LayerVector& bias_gradient);
  void DoActivationGradient(const size_t m, const size_t n, const LayerMatrix& upstream, const Activation activation,
                            const LayerMatrix& pre, const LayerMatrix& c, const LayerVector& bias_gradient,
                            const LayerGroups& groups);
  void DoGemmGrouped(const Transpose b_transpose, const size_t m, const size_t n, const size_t k, const float alpha,
                     const LayerMatrix& a, const LayerMatrix& b, const size_t b_stride, const LayerVector& bias,
                     const Activation activation, const LayerMatrix& pre, const float beta, const LayerMatrix& c,
                     const LayerGroups& groups);
  void DoGemmGroupedGradient(const size_t m, const size_t n, const size_t k, const float alpha, const LayerMatrix& a,
                             const LayerMatrix& b, const float beta, const LayerMatrix& c, const size_t c_stride,
                             const LayerGroups& groups);

 private:
  void Launch(clbh_layer_desc& desc);
};

// =================================================================================================
}  // namespace clblast

#endif  // CLBLAST_HIP_ROUTINES_XLAYER_HPP_
