// Calls of the layer products that the argument checks (clblast_amd/csrc/routines/xlayer.cpp) have to tell apart, without a GPU: the
// device layer is replaced by buffers of given sizes - nobody looks inside them, so that they can be as large as the largest
// calls need - and a launch that keeps the descriptor. Compiled and run by tests/test_layer_limits_cpu.py.
#include <cstdio>
#include <initializer_list>
#include <vector>

#include "routines/xlayer.hpp"

using namespace clblast;

namespace {
struct Extent { size_t begin, bytes; };
std::vector<Extent> buffers;
int launches = 0, violations = 0;
clbh_layer_desc last{};
}  // namespace

extern "C" {
int clbh_stream_device(hipStream_t, int* device) { *device = 0; return 0; }
int clbh_stream_is_alias(hipStream_t) { return 0; }
int clbh_stream_capturing(hipStream_t, int* capturing) { *capturing = 0; return 0; }
int clbh_buffer_extent(const void* pointer, size_t* available) {
  const size_t at = reinterpret_cast<size_t>(pointer);
  for (const auto& b : buffers) { if (at >= b.begin && at - b.begin < b.bytes) { *available = b.begin + b.bytes - at; return 0; } }
  return 1;
}
int clbh_event_record(hipEvent_t, hipStream_t) { return 0; }
int clbh_alloc(void** pointer, size_t bytes) { *pointer = ::operator new(bytes); return 0; }
int clbh_free(void* pointer) { ::operator delete(pointer); return 0; }
int clbh_alloc_async(void** pointer, size_t bytes, hipStream_t) { return clbh_alloc(pointer, bytes); }
int clbh_free_async(void* pointer, hipStream_t) { return clbh_free(pointer); }
const char* clbh_error_string(int) { return "refused"; }
int clbh_compute_units(int* units) { *units = 256; return 0; }
size_t clbh_gemm_workspace_bytes(const clbh_gemm_desc*) { return 0; }
int clbh_gemm_workspace_optional(const clbh_gemm_desc*) { return 0; }
int clbh_gemm_launch(const clbh_gemm_desc*, hipStream_t) { return 0; }
int clbh_copy_matrix(int, int, int, const void*, long long, long long, void*, long long, long long, hipStream_t) { return 0; }
size_t clbh_layer_workspace_bytes(const clbh_layer_desc*) { return 0; }
int clbh_layer_launch(const clbh_layer_desc* d, hipStream_t) { ++launches; last = *d; return 0; }
}  // extern "C"

namespace {
hipStream_t stream = nullptr;

template <typename T, typename F>
void Code(const StatusCode expected, const char* what, F&& body) {
  const int before = launches;
  auto status = StatusCode::kSuccess;
  try { auto routine = Xlayer<T>(&stream, nullptr); body(routine); } catch (...) { status = DispatchException(true); }
  if (status != expected || (status == StatusCode::kSuccess) != (launches == before + 1)) {
    ++violations;
    std::printf("VIOLATION %s: %d instead of %d\n", what, static_cast<int>(status), static_cast<int>(expected));
  }
}

const void* Place(const size_t bytes) {
  const size_t begin = buffers.empty() ? size_t{1} << 40 : buffers.back().begin + buffers.back().bytes + 4096;
  buffers.push_back({begin / 256 * 256 + 256, bytes});
  return reinterpret_cast<const void*>(buffers.back().begin);
}

// One call of m x n x k whose buffers are as large as it needs, and whether it is accepted
template <typename T>
void Reach(const bool accepted, const char* what, const size_t m, const size_t n, const size_t k, const bool a_turned, const bool b_turned) {
  const LayerMatrix a{Place(m * k * sizeof(T)), 0, a_turned ? m : k}, b{Place(n * k * sizeof(T)), 0, b_turned ? k : n}, c{Place(m * n * sizeof(T)), 0, n};
  const auto turn = [](const bool turned) { return turned ? Transpose::kYes : Transpose::kNo; };
  Code<T>(accepted ? StatusCode::kSuccess : StatusCode::kInvalidDimension, what, [&](Xlayer<T>& r) {
    r.DoGemmEpilogue(turn(a_turned), turn(b_turned), m, n, k, 1.0f, a, b, LayerVector{nullptr, 0, 0}, Activation::kNone, LayerMatrix{nullptr, 0, 0}, 0.0f,
                     LayerMatrix{nullptr, 0, 0}, c);
  });
}

// Rows of a matrix, or depths of a transposed one, further apart than 32-bit offsets reach over a slab's lines
void FarLines() {
  constexpr size_t kMost16 = 143165559, kMost32 = 71582779;  // 15 lines of 16- and 32-bit elements and a piece: 2^32 bytes
  Reach<half>(true, "16 rows", 16, 3, kMost16 / 8 * 8, false, true);
  Reach<half>(false, "16 rows, one piece more", 16, 3, kMost16 + 8, false, true);
  Reach<half>(false, "16 features", 3, 16, kMost16 + 8, false, true);
  Reach<half>(false, "any rows", 5000, 1, 2000000000, false, true);
  Reach<half>(true, "a row alone", 1, 1, (size_t{1} << 31) - 1024, false, true);
  Reach<bfloat16>(true, "two rows", 2, 2, (size_t{1} << 31) - 1024, false, true);
  Reach<float>(true, "16 rows of fp32", 16, 3, kMost32 / 8 * 8, false, true);
  Reach<float>(false, "16 rows of fp32, one piece more", 16, 3, kMost32 + 8, false, true);
  Reach<float>(false, "two rows of fp32", 2, 1, (size_t{1} << 31) - 1024, false, true);
  Reach<float>(true, "a row of fp32 alone", 1, 1, (size_t{1} << 31) - 1024, false, true);
  Reach<half>(true, "depths of 300 million features", 1, 300000000, 2, false, false);
  Reach<half>(false, "depths of 310 million features", 1, 310000000, 2, false, false);
  Reach<half>(false, "depths of 310 million rows", 310000000, 1, 2, true, true);
  Reach<half>(true, "many rows, not transposed", (size_t{1} << 31) - 1024, 1, 2, false, true);
  Reach<half>(true, "a long depth of few rows and features", 7, 9, (size_t{1} << 31) - 1024, true, false);
}

// One bias for all groups, as one matrix for all of them: it is only read
void SharedBias() {
  const LayerMatrix a{Place(10 * 14 * 2), 0, 14}, b{Place(3 * 14 * 12 * 2), 0, 12}, c{Place(10 * 12 * 2), 0, 12}, nothing{nullptr, 0, 0};
  const void* bias = Place(12 * 2);
  const LayerGroups groups{3, Place(4 * 8), 0};
  const auto call = [&](const StatusCode code, const char* what, const size_t offset, const size_t stride) {
    Code<half>(code, what, [&](Xlayer<half>& r) {
      r.DoGemmGrouped(Transpose::kNo, 10, 12, 14, 1.0f, a, b, 14 * 12, LayerVector{bias, offset, stride}, Activation::kNone, nothing, 0.0f, c, groups);
    });
  };
  call(StatusCode::kSuccess, "one bias for all groups", 0, 0);
  if (last.bias != bias || last.bias_stride != 0) { ++violations; std::printf("VIOLATION the shared bias\n"); }
  call(StatusCode::kInsufficientMemoryX, "one bias for all groups, short", 1, 0);
  call(StatusCode::kInvalidIncrementX, "biases that overlap", 0, 11);
  call(StatusCode::kInsufficientMemoryX, "a bias for every group", 0, 12);
}
}  // namespace

int main() {
  FarLines();
  SharedBias();
  std::printf("launches %d violations %d\n", launches, violations);
  return violations == 0 ? 0 : 1;
}
