// =================================================================================================
// Xlayer<T> host logic (see xlayer.hpp).
// =================================================================================================
#include "routines/xlayer.hpp"

#include <memory>

#include "device/layer_plans.hpp"

namespace clblast {
// =================================================================================================
namespace {

template <typename T> constexpr int LayerType();
template <> constexpr int LayerType<half>() { return CLBH_TYPE_FP16; }
template <> constexpr int LayerType<bfloat16>() { return CLBH_TYPE_BF16; }
template <> constexpr int LayerType<float>() { return CLBH_TYPE_FP32; }

void TestSizes(const size_t m, const size_t n, const size_t k) {
  constexpr auto kLimit = static_cast<size_t>(CLBH_LAYER_MAX_SIZE);
  if (m == 0 || n == 0 || k == 0) { throw BLASError(StatusCode::kInvalidDimension); }
  if (m > kLimit || n > kLimit || k > kLimit) { throw BLASError(StatusCode::kInvalidDimension, "dimension exceeds 2^31 - 1024"); }
}

void TestActivation(const Activation activation) {
  switch (activation) {
    case Activation::kNone:
    case Activation::kRelu:
    case Activation::kGelu:
    case Activation::kGeluTanh:
    case Activation::kSilu: return;
  }
  throw BLASError(StatusCode::kInvalidValue, "unknown activation");
}

void TestTranspose(const Transpose transpose) {
  if (transpose != Transpose::kNo && transpose != Transpose::kYes && transpose != Transpose::kConjugate) {
    throw BLASError(StatusCode::kInvalidValue, "unknown transpose");
  }
}

// Bytes from a pointer to the end of its allocation
size_t Available(const void* pointer, const StatusCode bad_buffer) {
  auto available = size_t{0};
  if (pointer == nullptr || clbh_buffer_extent(pointer, &available) != 0) { throw BLASError(bad_buffer); }
  return available;
}

// `rows` rows of `cols` elements at distance ld (and `count` such matrices at distance stride): the contract of the GEMM
// routines' matrix tests - leading dimension, buffer, size - without overflow in the sizes
void TestMatrix(const size_t rows, const size_t cols, const LayerMatrix& matrix, const size_t element, const StatusCode bad_ld,
                const StatusCode too_small, const StatusCode bad_buffer, const size_t count = 1, const size_t stride = 0) {
  if (matrix.ld < cols) { throw BLASError(bad_ld); }
  const auto available = Available(matrix.pointer, bad_buffer);
  if (reinterpret_cast<size_t>(matrix.pointer) % element != 0) { throw BLASError(bad_buffer, "unaligned pointer"); }
  const auto last = static_cast<unsigned __int128>(matrix.ld) * (rows - 1) + static_cast<unsigned __int128>(stride) * (count - 1) + cols + matrix.offset;
  if (last * element > available) { throw BLASError(too_small); }
}
void TestA(const size_t rows, const size_t cols, const LayerMatrix& matrix, const size_t element) {
  TestMatrix(rows, cols, matrix, element, StatusCode::kInvalidLeadDimA, StatusCode::kInsufficientMemoryA, StatusCode::kInvalidMatrixA);
}
void TestB(const size_t rows, const size_t cols, const LayerMatrix& matrix, const size_t element, const size_t count = 1,
           const size_t stride = 0) {
  TestMatrix(rows, cols, matrix, element, StatusCode::kInvalidLeadDimB, StatusCode::kInsufficientMemoryB, StatusCode::kInvalidMatrixB, count, stride);
}
void TestC(const size_t rows, const size_t cols, const LayerMatrix& matrix, const size_t element, const size_t count = 1,
           const size_t stride = 0) {
  TestMatrix(rows, cols, matrix, element, StatusCode::kInvalidLeadDimC, StatusCode::kInsufficientMemoryC, StatusCode::kInvalidMatrixC, count, stride);
}
// (stride 0: one vector, read for every group. The sums of groups are given their n as a stride.)
void TestVector(const size_t n, const LayerVector& vector, const size_t count, const size_t element) {
  if (vector.stride != 0 && vector.stride < n && count > 1) { throw BLASError(StatusCode::kInvalidIncrementX, "vectors of the groups overlap"); }
  TestMatrix(1, n, LayerMatrix{vector.pointer, vector.offset, n}, element, StatusCode::kInvalidIncrementX,
             StatusCode::kInsufficientMemoryX, StatusCode::kInvalidVectorX, count, vector.stride);
}
void TestGroups(const LayerGroups& groups, const size_t rows) {
  if (groups.count == 0 || groups.count > static_cast<size_t>(CLBH_LAYER_MAX_GROUPS)) { throw BLASError(StatusCode::kInvalidBatchCount); }
  if (rows >= static_cast<size_t>(CLBH_LAYER_MAX_GROUPED)) { throw BLASError(StatusCode::kInvalidDimension, "rows of a grouped call"); }
}
void TestOffsets(const LayerGroups& groups) {
  TestMatrix(1, groups.count + 1, LayerMatrix{groups.offsets, groups.offset, groups.count + 1}, sizeof(long long),
             StatusCode::kInvalidIncrementY, StatusCode::kInsufficientMemoryY, StatusCode::kInvalidVectorY);
}

template <typename T>
void* At(const LayerMatrix& matrix) {
  return (matrix.pointer == nullptr) ? nullptr : static_cast<char*>(const_cast<void*>(matrix.pointer)) + matrix.offset * sizeof(T);
}
template <typename T>
void* At(const LayerVector& vector) { return At<T>(LayerMatrix{vector.pointer, vector.offset, 0}); }
const long long* At(const LayerGroups& groups) { return static_cast<const long long*>(groups.offsets) + groups.offset; }

template <typename T>
clbh_layer_desc Describe(const size_t rows, const size_t features, const size_t depth, const float alpha, const Activation activation) {
  auto desc = clbh_layer_desc{};
  desc.type = LayerType<T>();
  desc.tile_variant = -1;
  desc.m = static_cast<int>(features);
  desc.n = static_cast<int>(rows);
  desc.k = static_cast<int>(depth);
  desc.alpha = alpha;
  desc.activation = static_cast<int>(activation);
  return desc;
}
template <typename T>
void SetC(clbh_layer_desc& desc, const LayerMatrix& c) { desc.c = At<T>(c); desc.c_ld = static_cast<long long>(c.ld); }
template <typename T>
void SetPre(clbh_layer_desc& desc, const LayerMatrix& pre) { desc.pre = At<T>(pre); desc.pre_ld = static_cast<long long>(pre.ld); }
// The caller's B holds the weights: the device layer's A. Its A holds the rows: the device layer's B.
template <typename T>
void SetOperands(clbh_layer_desc& desc, const LayerMatrix& a, const bool a_transposed, const LayerMatrix& b, const bool b_transposed) {
  desc.a = At<T>(b);
  desc.a_ld = static_cast<long long>(b.ld);
  desc.a_kcontig = b_transposed ? 1 : 0;
  desc.b = At<T>(a);
  desc.b_ld = static_cast<long long>(a.ld);
  desc.b_kcontig = a_transposed ? 0 : 1;
}

}  // namespace

template <typename T>
Xlayer<T>::Xlayer(hipStream_t* queue, hipEvent_t* event) : GemmRoutineBase(queue, event, Precision::kSingle) {}

template <typename T>
void Xlayer<T>::DoGemmEpilogue(const Transpose a_transpose, const Transpose b_transpose, const size_t m, const size_t n,
                               const size_t k, const float alpha, const LayerMatrix& a, const LayerMatrix& b,
                               const LayerVector& bias, const Activation activation, const LayerMatrix& pre, const float beta,
                               const LayerMatrix& residual, const LayerMatrix& c) {
  TestSizes(m, n, k);
  TestTranspose(a_transpose);
  TestTranspose(b_transpose);
  TestActivation(activation);
  const bool a_turned = a_transpose != Transpose::kNo, b_turned = b_transpose != Transpose::kNo;
  TestA(a_turned ? k : m, a_turned ? m : k, a, sizeof(T));
  TestB(b_turned ? n : k, b_turned ? k : n, b, sizeof(T));
  TestC(m, n, c, sizeof(T));
  if (pre.pointer != nullptr) { TestC(m, n, pre, sizeof(T)); }
  if (beta != 0.0f) { TestC(m, n, residual, sizeof(T)); }
  if (bias.pointer != nullptr) { TestVector(n, bias, 1, sizeof(T)); }
  auto desc = Describe<T>(m, n, k, alpha, activation);
  SetOperands<T>(desc, a, a_turned, b, b_turned);
  SetC<T>(desc, c);
  SetPre<T>(desc, pre);
  desc.bias = At<T>(bias);
  desc.beta = beta;
  if (beta != 0.0f) {
    desc.residual = At<T>(residual);
    desc.residual_ld = static_cast<long long>(residual.ld);
  }
  Launch(desc);
}

template <typename T>
void Xlayer<T>::DoGemmActivationGradient(const Transpose a_transpose, const Transpose b_transpose, const size_t m, const size_t n,
                                         const size_t k, const float alpha, const LayerMatrix& a, const LayerMatrix& b,
                                         const Activation activation, const LayerMatrix& pre, const LayerMatrix& c,
                                         const LayerVector& bias_gradient) {
  TestSizes(m, n, k);
  TestTranspose(a_transpose);
  TestTranspose(b_transpose);
  TestActivation(activation);
  const bool a_turned = a_transpose != Transpose::kNo, b_turned = b_transpose != Transpose::kNo;
  TestA(a_turned ? k : m, a_turned ? m : k, a, sizeof(T));
  TestB(b_turned ? n : k, b_turned ? k : n, b, sizeof(T));
  TestC(m, n, c, sizeof(T));
  if (activation != Activation::kNone) { TestC(m, n, pre, sizeof(T)); }  // (the slope of none does not depend on Z)
  if (bias_gradient.pointer != nullptr) { TestVector(n, bias_gradient, 1, sizeof(T)); }
  auto desc = Describe<T>(m, n, k, alpha, activation);
  SetOperands<T>(desc, a, a_turned, b, b_turned);
  SetC<T>(desc, c);
  if (activation != Activation::kNone) { SetPre<T>(desc, pre); }
  desc.gradient = 1;
  desc.bias_gradient = At<T>(bias_gradient);
  Launch(desc);
}

template <typename T>
void Xlayer<T>::DoActivationGradient(const size_t m, const size_t n, const LayerMatrix& upstream, const Activation activation,
                                     const LayerMatrix& pre, const LayerMatrix& c, const LayerVector& bias_gradient,
                                     const LayerGroups& groups) {
  const bool grouped = groups.offsets != nullptr;
  if (grouped) { TestGroups(groups, m); }
  TestSizes(m, n, 1);
  TestActivation(activation);
  TestA(m, n, upstream, sizeof(T));
  if (activation != Activation::kNone) { TestB(m, n, pre, sizeof(T)); }
  if (c.pointer == nullptr && bias_gradient.pointer == nullptr) { throw BLASError(StatusCode::kInvalidMatrixC, "no output"); }
  if (c.pointer != nullptr) { TestC(m, n, c, sizeof(T)); }
  const auto count = grouped ? groups.count : size_t{1};
  if (bias_gradient.pointer != nullptr) { TestVector(n, LayerVector{bias_gradient.pointer, bias_gradient.offset, n}, count, sizeof(T)); }
  if (grouped) { TestOffsets(groups); }
  auto desc = Describe<T>(m, n, 1, 1.0f, activation);
  desc.upstream = At<T>(upstream);
  desc.upstream_ld = static_cast<long long>(upstream.ld);
  SetC<T>(desc, c);
  if (activation != Activation::kNone) { SetPre<T>(desc, pre); }
  desc.gradient = 1;
  desc.bias_gradient = At<T>(bias_gradient);
  if (grouped) {
    desc.grouping = CLBH_GROUPS_BY_ROWS;
    desc.groups = static_cast<int>(groups.count);
    desc.offsets = At(groups);
  }
  Launch(desc);
}

template <typename T>
void Xlayer<T>::DoGemmGrouped(const Transpose b_transpose, const size_t m, const size_t n, const size_t k, const float alpha,
                              const LayerMatrix& a, const LayerMatrix& b, const size_t b_stride, const LayerVector& bias,
                              const Activation activation, const LayerMatrix& pre, const float beta, const LayerMatrix& c,
                              const LayerGroups& groups) {
  TestGroups(groups, m);
  TestSizes(m, n, k);
  TestTranspose(b_transpose);
  TestActivation(activation);
  const bool b_turned = b_transpose != Transpose::kNo;
  TestA(m, k, a, sizeof(T));
  TestB(b_turned ? n : k, b_turned ? k : n, b, sizeof(T), groups.count, b_stride);
  TestC(m, n, c, sizeof(T));
  if (pre.pointer != nullptr) { TestC(m, n, pre, sizeof(T)); }
  if (bias.pointer != nullptr) { TestVector(n, bias, groups.count, sizeof(T)); }
  TestOffsets(groups);
  auto desc = Describe<T>(m, n, k, alpha, activation);
  SetOperands<T>(desc, a, false, b, b_turned);
  desc.a_stride = static_cast<long long>(b_stride);
  SetC<T>(desc, c);
  SetPre<T>(desc, pre);
  desc.bias = At<T>(bias);
  desc.bias_stride = static_cast<long long>(bias.stride);
  desc.beta = beta;
  desc.residual = desc.c;
  desc.residual_ld = desc.c_ld;
  desc.grouping = CLBH_GROUPS_BY_ROWS;
  desc.groups = static_cast<int>(groups.count);
  desc.offsets = At(groups);
  Launch(desc);
}

template <typename T>
void Xlayer<T>::DoGemmGroupedGradient(const size_t m, const size_t n, const size_t k, const float alpha, const LayerMatrix& a,
                                      const LayerMatrix& b, const float beta, const LayerMatrix& c, const size_t c_stride,
                                      const LayerGroups& groups) {
  TestGroups(groups, k);
  TestSizes(m, n, k);
  TestA(k, m, a, sizeof(T));
  TestB(k, n, b, sizeof(T));
  if (c.ld >= n && groups.count > 1) {  // one behind the other, or side by side within the rows
    using Wide = unsigned __int128;
    const bool behind = c_stride >= static_cast<Wide>(m - 1) * c.ld + n;
    const bool beside = c_stride >= n && static_cast<Wide>(groups.count - 1) * c_stride + n <= c.ld;
    if (!behind && !beside) { throw BLASError(StatusCode::kInvalidLeadDimC, "results of the groups overlap"); }
  }
  TestC(m, n, c, sizeof(T), groups.count, c_stride);
  TestOffsets(groups);
  auto desc = Describe<T>(m, n, k, alpha, Activation::kNone);
  SetOperands<T>(desc, a, true, b, false);
  SetC<T>(desc, c);
  desc.c_stride = static_cast<long long>(c_stride);
  desc.beta = beta;
  desc.residual = desc.c;
  desc.residual_ld = desc.c_ld;
  desc.grouping = CLBH_GROUPS_BY_DEPTH;
  desc.groups = static_cast<int>(groups.count);
  desc.offsets = At(groups);
  Launch(desc);
}

template <typename T>
void Xlayer<T>::Launch(clbh_layer_desc& desc) {
  if (!clbh::LayerOperandsReachable(desc)) { throw BLASError(StatusCode::kInvalidDimension, "rows of an operand are too long"); }
  ApplyLayerOverrides(sizeof(T) == 4 ? Precision::kSingle : Precision::kHalf, desc.tile_variant, desc.split_k);
  std::unique_ptr<StreamScratch> scratch;
  desc.workspace_bytes = clbh_layer_workspace_bytes(&desc);
  if (desc.workspace_bytes > 0) {
    scratch.reset(new StreamScratch(desc.workspace_bytes, stream(), "partial sums"));
    desc.workspace = scratch->get();
  }
  CheckDevice(clbh_layer_launch(&desc, stream()), "clbh_layer_launch");
  Finish();
}

template class Xlayer<half>;
template class Xlayer<float>;
template class Xlayer<bfloat16>;

// =================================================================================================
}  // namespace clblast
