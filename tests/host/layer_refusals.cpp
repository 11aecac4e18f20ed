// The argument checks of the layer products (clblast_amd/csrc/routines/xlayer.cpp) without a GPU: the device layer is
// replaced by a few buffers of known sizes and by a launch that recomputes, for every accepted call, the last byte that each
// operand reaches and checks that it lies inside its buffer. Compiled and run by tests/test_layers_cpu.py.
#include <cstdio>
#include <cstring>
#include <vector>

#include "routines/xlayer.hpp"

using namespace clblast;

namespace {
struct Fake { char* begin; size_t bytes; };
std::vector<Fake> buffers;
int launches = 0, failures = 0;
bool refuse_workspace = false;

bool Inside(const void* first, const long long bytes) {
  const char* at = static_cast<const char*>(first);
  for (const auto& b : buffers) { if (at >= b.begin && at + bytes <= b.begin + b.bytes) { return true; } }
  return false;
}
void Expect(const bool ok, const char* what) { if (!ok) { ++failures; std::printf("VIOLATION %s\n", what); } }
}  // namespace

extern "C" {
int clbh_stream_device(hipStream_t, int* device) { *device = 0; return 0; }
int clbh_stream_is_alias(hipStream_t) { return 0; }
int clbh_stream_capturing(hipStream_t, int* capturing) { *capturing = 0; return 0; }
int clbh_buffer_extent(const void* pointer, size_t* available) {
  const char* at = static_cast<const char*>(pointer);
  for (const auto& b : buffers) { if (at >= b.begin && at < b.begin + b.bytes) { *available = static_cast<size_t>(b.begin + b.bytes - at); return 0; } }
  return 1;
}
int clbh_event_record(hipEvent_t, hipStream_t) { return 0; }
int clbh_alloc(void** pointer, size_t bytes) { if (refuse_workspace) { return 2; } *pointer = ::operator new(bytes); return 0; }
int clbh_free(void* pointer) { ::operator delete(pointer); return 0; }
int clbh_alloc_async(void** pointer, size_t bytes, hipStream_t) { return clbh_alloc(pointer, bytes); }
int clbh_free_async(void* pointer, hipStream_t) { return clbh_free(pointer); }
const char* clbh_error_string(int) { return "refused"; }
int clbh_compute_units(int* units) { *units = 256; return 0; }
size_t clbh_gemm_workspace_bytes(const clbh_gemm_desc*) { return 0; }
int clbh_gemm_workspace_optional(const clbh_gemm_desc*) { return 0; }
int clbh_gemm_launch(const clbh_gemm_desc*, hipStream_t) { return 0; }
int clbh_copy_matrix(int, int, int, const void*, long long, long long, void*, long long, long long, hipStream_t) { return 0; }
size_t clbh_layer_workspace_bytes(const clbh_layer_desc* d) { return d->gradient ? 1024 : 0; }
int clbh_layer_launch(const clbh_layer_desc* d, hipStream_t) {
  ++launches;
  const long long size = d->type == CLBH_TYPE_FP32 ? 4 : 2;
  const auto matrix = [&](const void* p, const long long lines, const long long length, const long long ld) {
    return Inside(p, ((lines - 1) * ld + length) * size);
  };
  const long long groups = d->grouping == CLBH_GROUPS_NONE ? 1 : d->groups;
  if (d->upstream != nullptr) { Expect(matrix(d->upstream, d->n, d->m, d->upstream_ld), "upstream"); }
  else {
    const long long matrices = d->grouping == CLBH_GROUPS_BY_ROWS ? groups : 1;
    Expect(matrix(static_cast<const char*>(d->a) + (matrices - 1) * d->a_stride * size, d->a_kcontig ? d->m : d->k, d->a_kcontig ? d->k : d->m, d->a_ld), "a");
    Expect(matrix(d->b, d->b_kcontig ? d->n : d->k, d->b_kcontig ? d->k : d->n, d->b_ld), "b");
    Expect(d->c != nullptr, "c");
  }
  if (d->c != nullptr) {
    const long long results = d->grouping == CLBH_GROUPS_BY_DEPTH ? groups : 1;
    Expect(matrix(static_cast<char*>(d->c) + (results - 1) * d->c_stride * size, d->n, d->m, d->c_ld), "c");
  }
  if (d->pre != nullptr) { Expect(matrix(d->pre, d->n, d->m, d->pre_ld), "pre"); }
  if (d->beta != 0.0f) { Expect(d->residual != nullptr && matrix(d->residual, d->n, d->m, d->residual_ld), "residual"); }
  if (d->bias != nullptr) { Expect(Inside(static_cast<const char*>(d->bias) + (groups - 1) * d->bias_stride * size, d->m * size), "bias"); }
  if (d->bias_gradient != nullptr) { Expect(Inside(d->bias_gradient, (d->grouping == CLBH_GROUPS_BY_ROWS ? groups : 1) * d->m * size), "bias_gradient"); }
  if (d->offsets != nullptr) { Expect(Inside(d->offsets, (d->groups + 1) * 8), "offsets"); }
  return 0;
}
}  // extern "C"

namespace {
hipStream_t stream = nullptr;
template <typename F>
void Code(const StatusCode expected, const char* what, F&& body) {
  const int before = launches;
  auto status = StatusCode::kSuccess;
  try { auto routine = Xlayer<half>(&stream, nullptr); body(routine); } catch (...) { status = DispatchException(true); }
  if (status != expected) { ++failures; std::printf("VIOLATION %s: %d instead of %d\n", what, static_cast<int>(status), static_cast<int>(expected)); }
  if ((status == StatusCode::kSuccess) != (launches == before + 1)) { ++failures; std::printf("VIOLATION %s: launched or not\n", what); }
}
}  // namespace

int main() {
  const auto make = [](const size_t bytes) { buffers.push_back({static_cast<char*>(::operator new(bytes)), bytes}); return static_cast<void*>(buffers.back().begin); };
  // m = 10 rows, n = 12, k = 14; every buffer exactly as large as the call needs
  void* a = make(10 * 14 * 2);
  void* b = make(14 * 12 * 2);
  void* c = make(10 * 12 * 2);
  void* pre = make(10 * 12 * 2);
  void* bias = make(12 * 2);
  void* tiny = make(2);
  void* experts = make(3 * 14 * 12 * 2);
  void* offsets = make(4 * 8);
  void* sums = make(3 * 12 * 2);
  void* weights = make(3 * 14 * 12 * 2);
  const LayerVector none{nullptr, 0, 0};
  const LayerMatrix nothing{nullptr, 0, 0};
  const LayerGroups three{3, offsets, 0}, ungrouped{1, nullptr, 0};
  const auto no = Transpose::kNo, yes = Transpose::kYes;
  const auto gelu = Activation::kGelu;

  const auto epilogue = [&](const StatusCode code, const char* what, const LayerMatrix& A, const LayerMatrix& B, const LayerVector& bs, const LayerMatrix& P,
                            const float beta, const LayerMatrix& R, const LayerMatrix& C, const size_t m = 10, const size_t n = 12, const size_t k = 14,
                            const Transpose ta = Transpose::kNo, const Activation act = Activation::kGelu) {
    Code(code, what, [&](Xlayer<half>& r) { r.DoGemmEpilogue(ta, Transpose::kNo, m, n, k, 1.0f, A, B, bs, act, P, beta, R, C); });
  };
  const LayerMatrix A{a, 0, 14}, B{b, 0, 12}, C{c, 0, 12}, P{pre, 0, 12};
  const LayerVector V{bias, 0, 0};
  epilogue(StatusCode::kSuccess, "all fits", A, B, V, P, 1.0f, C, C);
  epilogue(StatusCode::kSuccess, "residual not looked at", A, B, none, nothing, 0.0f, LayerMatrix{reinterpret_cast<void*>(3), 9, 1}, C);
  epilogue(StatusCode::kSuccess, "a transposed", LayerMatrix{a, 0, 10}, B, V, P, 0.0f, nothing, C, 10, 12, 14, yes);
  epilogue(StatusCode::kInvalidDimension, "m = 0", A, B, V, P, 0.0f, nothing, C, 0);
  epilogue(StatusCode::kInvalidDimension, "n = 0", A, B, V, P, 0.0f, nothing, C, 10, 0);
  epilogue(StatusCode::kInvalidDimension, "k = 0", A, B, V, P, 0.0f, nothing, C, 10, 12, 0);
  epilogue(StatusCode::kInvalidDimension, "m too large", A, B, V, P, 0.0f, nothing, C, size_t{1} << 32);
  for (const auto size : {size_t{0x7fffffff}, (size_t{1} << 31) - 1023}) {  // a tile that begins inside would end beyond 32 bits
    epilogue(StatusCode::kInvalidDimension, "m close to 2^31", A, B, V, P, 0.0f, nothing, C, size);
    epilogue(StatusCode::kInvalidDimension, "n close to 2^31", A, B, V, P, 0.0f, nothing, C, 10, size);
    epilogue(StatusCode::kInvalidDimension, "k close to 2^31", A, B, V, P, 0.0f, nothing, C, 10, 12, size);
  }
  epilogue(StatusCode::kInvalidValue, "activation", A, B, V, P, 0.0f, nothing, C, 10, 12, 14, no, static_cast<Activation>(7));
  epilogue(StatusCode::kInvalidValue, "transpose", A, B, V, P, 0.0f, nothing, C, 10, 12, 14, static_cast<Transpose>(1));
  epilogue(StatusCode::kInvalidLeadDimA, "a_ld", LayerMatrix{a, 0, 13}, B, V, P, 0.0f, nothing, C);
  epilogue(StatusCode::kInvalidLeadDimB, "b_ld", A, LayerMatrix{b, 0, 11}, V, P, 0.0f, nothing, C);
  epilogue(StatusCode::kInvalidLeadDimC, "c_ld", A, B, V, P, 0.0f, nothing, LayerMatrix{c, 0, 11});
  epilogue(StatusCode::kInvalidLeadDimC, "pre_ld", A, B, V, LayerMatrix{pre, 0, 11}, 0.0f, nothing, C);
  epilogue(StatusCode::kInvalidLeadDimC, "residual_ld", A, B, V, P, 1.0f, LayerMatrix{c, 0, 11}, C);
  epilogue(StatusCode::kInsufficientMemoryA, "a short", LayerMatrix{a, 1, 14}, B, V, P, 0.0f, nothing, C);
  epilogue(StatusCode::kInsufficientMemoryA, "a_ld overflows", LayerMatrix{a, 0, ~size_t{0} / 4}, B, V, P, 0.0f, nothing, C);
  epilogue(StatusCode::kInsufficientMemoryA, "a_offset overflows", LayerMatrix{a, ~size_t{0}, 14}, B, V, P, 0.0f, nothing, C);
  epilogue(StatusCode::kInsufficientMemoryB, "b short", A, LayerMatrix{b, 1, 12}, V, P, 0.0f, nothing, C);
  epilogue(StatusCode::kInsufficientMemoryC, "c short", A, B, V, P, 0.0f, nothing, LayerMatrix{c, 0, 13});
  epilogue(StatusCode::kInsufficientMemoryC, "pre short", A, B, V, LayerMatrix{pre, 2, 12}, 0.0f, nothing, C);
  epilogue(StatusCode::kInsufficientMemoryC, "residual short", A, B, V, P, 1.0f, LayerMatrix{c, 1, 12}, C);
  epilogue(StatusCode::kInsufficientMemoryX, "bias short", A, B, LayerVector{bias, 1, 0}, P, 0.0f, nothing, C);
  epilogue(StatusCode::kInvalidMatrixA, "a unknown", LayerMatrix{reinterpret_cast<void*>(64), 0, 14}, B, V, P, 0.0f, nothing, C);
  epilogue(StatusCode::kInvalidMatrixA, "a null", LayerMatrix{nullptr, 0, 14}, B, V, P, 0.0f, nothing, C);
  epilogue(StatusCode::kInvalidMatrixA, "a between elements", LayerMatrix{static_cast<char*>(a) + 1, 0, 14}, B, V, P, 0.0f, nothing, C, 9);
  epilogue(StatusCode::kInvalidMatrixC, "residual null", A, B, V, P, 1.0f, LayerMatrix{nullptr, 0, 12}, C);
  epilogue(StatusCode::kInvalidVectorX, "bias unknown", A, B, LayerVector{reinterpret_cast<void*>(64), 0, 0}, P, 0.0f, nothing, C);

  const auto gradient = [&](const StatusCode code, const char* what, const LayerMatrix& Z, const LayerVector& d, const Activation act) {
    Code(code, what, [&](Xlayer<half>& r) { r.DoGemmActivationGradient(no, no, 10, 12, 14, 1.0f, A, B, act, Z, C, d); });
  };
  gradient(StatusCode::kSuccess, "gradient", P, V, gelu);
  gradient(StatusCode::kSuccess, "gradient without an activation", nothing, V, Activation::kNone);
  gradient(StatusCode::kSuccess, "gradient without sums", P, none, gelu);
  gradient(StatusCode::kInvalidMatrixC, "gradient without Z", LayerMatrix{nullptr, 0, 12}, V, gelu);
  gradient(StatusCode::kInsufficientMemoryX, "bias gradient short", P, LayerVector{tiny, 0, 0}, gelu);
  refuse_workspace = true;
  ReleaseCachedScratch();
  gradient(StatusCode::kTempBufferAllocFailure, "no memory for the sums", P, V, gelu);
  refuse_workspace = false;

  const auto activation = [&](const StatusCode code, const char* what, const LayerMatrix& out, const LayerVector& d, const LayerGroups& g, const size_t m = 10) {
    Code(code, what, [&](Xlayer<half>& r) { r.DoActivationGradient(m, 12, C, gelu, P, out, d, g); });
  };
  activation(StatusCode::kSuccess, "activation", C, V, ungrouped);
  activation(StatusCode::kSuccess, "activation, sums alone", nothing, V, ungrouped);
  activation(StatusCode::kSuccess, "activation by group", C, LayerVector{sums, 0, 12}, three);
  activation(StatusCode::kInvalidMatrixC, "activation without an output", nothing, none, ungrouped);
  activation(StatusCode::kInsufficientMemoryX, "sums of the groups", C, V, three);
  activation(StatusCode::kInvalidBatchCount, "no groups", C, none, LayerGroups{0, offsets, 0});
  activation(StatusCode::kInsufficientMemoryY, "offsets short", C, none, LayerGroups{4, offsets, 0});
  activation(StatusCode::kInsufficientMemoryY, "offsets behind", C, none, LayerGroups{3, offsets, 1});
  activation(StatusCode::kInvalidVectorY, "offsets unaligned", C, none, LayerGroups{1, static_cast<char*>(offsets) + 4, 0});
  activation(StatusCode::kInvalidVectorY, "offsets unknown", C, none, LayerGroups{1, reinterpret_cast<void*>(64), 0});
  activation(StatusCode::kInvalidDimension, "rows of a grouped call", C, none, three, size_t{1} << 26);

  const auto grouped = [&](const StatusCode code, const char* what, const size_t stride, const LayerVector& bs, const LayerGroups& g, const size_t m = 10) {
    Code(code, what, [&](Xlayer<half>& r) { r.DoGemmGrouped(no, m, 12, 14, 1.0f, A, LayerMatrix{experts, 0, 12}, stride, bs, gelu, P, 0.5f, C, g); });
  };
  grouped(StatusCode::kSuccess, "grouped", 14 * 12, LayerVector{sums, 0, 12}, three);
  grouped(StatusCode::kSuccess, "grouped, one matrix", 0, none, three);
  grouped(StatusCode::kInsufficientMemoryB, "experts short", 14 * 12 + 1, none, three);
  grouped(StatusCode::kInsufficientMemoryB, "stride overflows", ~size_t{0} / 2, none, three);
  grouped(StatusCode::kInvalidIncrementX, "biases overlap", 14 * 12, LayerVector{sums, 0, 11}, three);
  grouped(StatusCode::kInvalidBatchCount, "too many groups", 0, none, LayerGroups{(size_t{1} << 16) + 1, offsets, 0});
  grouped(StatusCode::kInvalidVectorY, "no offsets", 0, none, LayerGroups{3, nullptr, 0});
  grouped(StatusCode::kInvalidDimension, "no rows", 0, none, three, 0);

  const auto depth = [&](const StatusCode code, const char* what, const size_t ld, const size_t stride, const size_t k = 10) {
    Code(code, what, [&](Xlayer<half>& r) { r.DoGemmGroupedGradient(14, 12, k, 1.0f, A, C, 0.0f, LayerMatrix{weights, 0, ld}, stride, three); });
  };
  depth(StatusCode::kSuccess, "grouped gradient", 12, 14 * 12);
  depth(StatusCode::kInvalidLeadDimC, "results overlap", 12, 13 * 12);
  depth(StatusCode::kInvalidLeadDimC, "results overlap by an element", 13, 13 * 13 + 11);
  depth(StatusCode::kSuccess, "results without the last row's padding", 12, 13 * 12 + 12);
  depth(StatusCode::kSuccess, "results side by side", 36, 12);
  depth(StatusCode::kInvalidLeadDimC, "results side by side overlap", 36, 11);
  depth(StatusCode::kInvalidLeadDimC, "results side by side reach the next row", 35, 12);
  depth(StatusCode::kInvalidLeadDimC, "stride of zero", 36, 0);
  depth(StatusCode::kInvalidLeadDimC, "c_ld", 11, 14 * 12);
  depth(StatusCode::kInsufficientMemoryC, "results short", 12, 14 * 12 + 1);
  depth(StatusCode::kInvalidDimension, "no depth", 12, 14 * 12, 0);

  Code(StatusCode::kSuccess, "queue", [&](Xlayer<half>& r) { r.DoGemmEpilogue(no, no, 10, 12, 14, 1.0f, A, B, none, gelu, nothing, 0.0f, nothing, C); });
  auto status = StatusCode::kSuccess;
  try { Xlayer<float>(nullptr, nullptr); } catch (...) { status = DispatchException(true); }
  Expect(status == StatusCode::kInvalidCommandQueue, "null queue");
  std::printf("launches %d violations %d\n", launches, failures);
  return failures == 0 ? 0 : 1;
}
