// C ABI of libilgpu_hip_algorithms.so: argument validation (mirroring the
// checks and exception kinds of the reference's host-side delegates) and
// dispatch to the kernel launchers.  No GPU work is enqueued when validation
// fails, and nothing here allocates device memory.
#include <atomic>
#include <cstring>
#include <mutex>
#include <string>
#include <vector>

#include "elements.hpp"
#include "kernels.hpp"
#include "operators.hpp"

namespace ilgpu_hip {

namespace {
thread_local int32_t g_last_runtime_error = 0;
std::atomic<int> g_cu_count[kMaxCachedDevices];
}  // namespace

void set_last_runtime_error(hipError_t e) { g_last_runtime_error = (int32_t)e; }

int current_device() {
  int dev = -1;
  return hipGetDevice(&dev) == hipSuccess ? dev : -1;
}

int device_cu_count() {
  const int dev = current_device();
  const bool cacheable = dev >= 0 && dev < kMaxCachedDevices;
  if (cacheable) {
    const int cached = g_cu_count[dev].load(std::memory_order_relaxed);
    if (cached > 0) return cached;
  }
  int cus = 0;
  if (dev < 0 ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) !=
          hipSuccess ||
      cus <= 0)
    cus = 256;
  if (cacheable) g_cu_count[dev].store(cus, std::memory_order_relaxed);
  return cus;
}

// ---- per-kernel timing ------------------------------------------------------
namespace {
struct ProfileRecord {
  const char* name;
  hipEvent_t start, stop;
};
struct ProfileTotal {
  std::string name;
  int64_t launches;
  double total_ms;
};
std::atomic<bool> g_profiling{false};
std::mutex g_profile_mutex;
std::vector<ProfileRecord> g_profile_pending;
std::vector<ProfileTotal> g_profile_totals;

// Waits for every pending event pair and folds it into the totals.
void drain_profile_records() {
  std::lock_guard<std::mutex> lock(g_profile_mutex);
  for (const ProfileRecord& r : g_profile_pending) {
    float ms = 0.0f;
    if (hipEventSynchronize(r.stop) == hipSuccess &&
        hipEventElapsedTime(&ms, r.start, r.stop) == hipSuccess) {
      ProfileTotal* t = nullptr;
      for (ProfileTotal& c : g_profile_totals)
        if (c.name == r.name) t = &c;
      if (t == nullptr) {
        g_profile_totals.push_back({r.name, 0, 0.0});
        t = &g_profile_totals.back();
      }
      t->launches += 1;
      t->total_ms += ms;
    }
    (void)hipEventDestroy(r.start);
    (void)hipEventDestroy(r.stop);
  }
  g_profile_pending.clear();
}
}  // namespace

ProfileScope::ProfileScope(hipStream_t stream, const char* name)
    : stream_(stream), name_(name), start_(nullptr), active_(false) {
  if (!g_profiling.load(std::memory_order_relaxed)) return;
  if (hipEventCreate(&start_) != hipSuccess) return;
  if (hipEventRecord(start_, stream_) != hipSuccess) {
    (void)hipEventDestroy(start_);
    return;
  }
  active_ = true;
}

ProfileScope::~ProfileScope() {
  if (!active_) return;
  hipEvent_t stop = nullptr;
  if (hipEventCreate(&stop) != hipSuccess ||
      hipEventRecord(stop, stream_) != hipSuccess) {
    (void)hipEventDestroy(start_);
    if (stop) (void)hipEventDestroy(stop);
    return;
  }
  std::lock_guard<std::mutex> lock(g_profile_mutex);
  g_profile_pending.push_back({name_, start_, stop});
}

namespace {

inline bool aligned_to(const void* p, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes) == 0;
}

// A view is valid when it has a buffer and a positive length
// (ArrayView.IsValid, ArrayView.cs:261-265).
inline bool valid_view(const void* p, int64_t length) {
  return p != nullptr && length > 0;
}

// The checks TempViewManager makes on the caller's ArrayView<int> temp
// (TempViewManager.cs:33-41, 84-89).
inline int32_t check_temp(const void* temp, int64_t temp_bytes,
                          int64_t required) {
  if (temp == nullptr || temp_bytes <= 0) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (!aligned_to(temp, 4)) return ILGPU_HIP_ERROR_UNALIGNED_TEMP;
  if (temp_bytes < required) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  return ILGPU_HIP_SUCCESS;
}

inline bool scan_reduce_type(int32_t t) {
  return t == ILGPU_HIP_I32 || t == ILGPU_HIP_I64 || t == ILGPU_HIP_U32 ||
         t == ILGPU_HIP_U64 || t == ILGPU_HIP_F32 || t == ILGPU_HIP_F64;
}

inline bool valid_op(int32_t op) {
  return op == ILGPU_HIP_OP_ADD || op == ILGPU_HIP_OP_MAX ||
         op == ILGPU_HIP_OP_MIN;
}

// A rows x columns matrix that a call reads (written = false) or writes.
inline int32_t check_matrix(const void* data, int64_t rows, int64_t columns, int64_t stride,
                            int elem_bytes, bool written) {
  if (columns == 0 || (rows > 0 && data == nullptr)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (rows < 0 || columns < 0 || stride < (written && rows > 1 ? columns : 0))
    return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (rows > INT32_MAX || columns > INT32_MAX || stride > INT32_MAX)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!aligned_to(data, elem_bytes)) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  return ILGPU_HIP_SUCCESS;
}

// The list of a norm or of a clip.
inline int32_t check_tensors(const ilgpu_hip_tensor* tensors, int64_t count) {
  if (count < 0) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (count > INT32_MAX) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (count > 0 && tensors == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  int64_t total = 0;
  for (int64_t k = 0; k < count; ++k) {
    const int eb = operator_elem_size(tensors[k].type);
    if (eb < 0) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
    if (tensors[k].length < 0) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
    if (tensors[k].length == 0) continue;
    if (tensors[k].data == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
    if (!aligned_to(tensors[k].data, eb)) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
    if (tensors[k].length > (INT64_C(1) << 40) - total) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
    total += tensors[k].length;
  }
  return ILGPU_HIP_SUCCESS;
}

}  // namespace
}  // namespace ilgpu_hip

using namespace ilgpu_hip;

extern "C" {

int32_t ilgpu_hip_version(void) { return ILGPU_HIP_ALGORITHMS_VERSION; }

const char* ilgpu_hip_status_string(int32_t status) {
  switch (status) {
    case ILGPU_HIP_SUCCESS: return "success";
    case ILGPU_HIP_ERROR_NULL_VIEW: return "invalid (null or empty) view";
    case ILGPU_HIP_ERROR_OUT_OF_RANGE: return "argument out of range";
    case ILGPU_HIP_ERROR_NOT_SUPPORTED: return "not supported";
    case ILGPU_HIP_ERROR_UNALIGNED_TEMP: return "unaligned temp allocation";
    case ILGPU_HIP_ERROR_RUNTIME: return "HIP runtime error";
    case ILGPU_HIP_ERROR_STATIC_LIMIT:
      return "input exceeds what the library's static scratch serves "
             "(ilgpu_hip_scan_static: 1 GiB of input)";
    default: return "unknown status";
  }
}

int32_t ilgpu_hip_last_runtime_error(void) { return g_last_runtime_error; }

int32_t ilgpu_hip_profile_enable(int32_t enabled) {
  drain_profile_records();
  if (enabled) {
    std::lock_guard<std::mutex> lock(g_profile_mutex);
    g_profile_totals.clear();
  }
  g_profiling.store(enabled != 0, std::memory_order_relaxed);
  return ILGPU_HIP_SUCCESS;
}

int32_t ilgpu_hip_profile_query(const char* kernel_name, int64_t* launches,
                                double* total_ms) {
  if (kernel_name == nullptr || launches == nullptr || total_ms == nullptr)
    return ILGPU_HIP_ERROR_NULL_VIEW;
  drain_profile_records();
  std::lock_guard<std::mutex> lock(g_profile_mutex);
  *launches = 0;
  *total_ms = 0.0;
  for (const ProfileTotal& t : g_profile_totals)
    if (t.name == kernel_name) {
      *launches = t.launches;
      *total_ms = t.total_ms;
    }
  return ILGPU_HIP_SUCCESS;
}

/* ---- radix sort -------------------------------------------------------- */

int32_t ilgpu_hip_radix_sort_temp_bytes(int64_t n, int32_t key_type,
                                        int32_t value_bytes,
                                        int64_t* temp_bytes) {
  if (temp_bytes == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  const int kb = elem_size(key_type);
  if (kb < 0) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (value_bytes != 0 && value_bytes != 1 && value_bytes != 2 &&
      value_bytes != 4 && value_bytes != 8 && value_bytes != 16)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (n < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (n > radix_sort_max_length()) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  *temp_bytes = radix_sort_temp_bytes(n, kb, value_bytes);
  return ILGPU_HIP_SUCCESS;
}

int32_t ilgpu_hip_radix_sort_temp_bytes_strided(int64_t n, int32_t key_type,
                                                int32_t value_bytes,
                                                int64_t key_stride,
                                                int64_t value_stride,
                                                int64_t* temp_bytes) {
  if (temp_bytes == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (key_stride < 1 || value_stride < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  const int32_t rc =
      ilgpu_hip_radix_sort_temp_bytes(n, key_type, value_bytes, temp_bytes);
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  *temp_bytes = radix_sort_temp_bytes(n, elem_size(key_type), value_bytes,
                                      key_stride, value_stride);
  return ILGPU_HIP_SUCCESS;
}

int32_t ilgpu_hip_radix_sort_keys(ilgpu_hip_stream_t stream, void* keys,
                                  int64_t n, int64_t stride, int32_t key_type,
                                  int32_t flags, void* temp,
                                  int64_t temp_bytes) {
  const int kb = elem_size(key_type);
  if (kb < 0) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!valid_view(keys, n)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (n > radix_sort_max_length()) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (stride < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (!aligned_to(keys, kb)) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (flags & ~(ILGPU_HIP_SORT_DESCENDING | ILGPU_HIP_SORT_FLOAT_TOTAL_ORDER))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  const int32_t rc = check_temp(temp, temp_bytes,
                                radix_sort_temp_bytes(n, kb, 0, stride, 1));
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  SortArgs a{keys, nullptr, stride, 1, n, key_type, 0, flags,
             ILGPU_HIP_VALUES_FROM_VIEW, temp};
  return launch_radix_sort(static_cast<hipStream_t>(stream), a);
}

int32_t ilgpu_hip_radix_sort_pairs(ilgpu_hip_stream_t stream, void* keys,
                                   int64_t key_stride, void* values,
                                   int64_t value_stride, int64_t n,
                                   int32_t key_type, int32_t value_bytes,
                                   int32_t flags, int32_t value_source,
                                   void* temp, int64_t temp_bytes) {
  const int kb = elem_size(key_type);
  if (kb < 0) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (value_bytes != 1 && value_bytes != 2 && value_bytes != 4 &&
      value_bytes != 8 && value_bytes != 16)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!valid_view(keys, n) || values == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (n > radix_sort_max_length()) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (key_stride < 1 || value_stride < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (!aligned_to(keys, kb) || !aligned_to(values, value_bytes))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (flags & ~(ILGPU_HIP_SORT_DESCENDING | ILGPU_HIP_SORT_FLOAT_TOTAL_ORDER))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (value_source != ILGPU_HIP_VALUES_FROM_VIEW &&
      value_source != ILGPU_HIP_VALUES_FROM_INDEX &&
      value_source != ILGPU_HIP_VALUES_FROM_INDEX_AS_FLOAT)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (value_source == ILGPU_HIP_VALUES_FROM_INDEX && value_bytes == 16)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (value_source == ILGPU_HIP_VALUES_FROM_INDEX_AS_FLOAT && value_bytes != 2 &&
      value_bytes != 4 && value_bytes != 8)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  const int32_t rc = check_temp(
      temp, temp_bytes,
      radix_sort_temp_bytes(n, kb, value_bytes, key_stride, value_stride));
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  SortArgs a{keys, values, key_stride, value_stride, n, key_type, value_bytes,
             flags, value_source, temp};
  return launch_radix_sort(static_cast<hipStream_t>(stream), a);
}

int32_t ilgpu_hip_selftest_lds_atomic_order(ilgpu_hip_stream_t stream,
                                            int32_t rows, int64_t* mismatches) {
  if (mismatches == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (rows < 1 || rows > (1 << 20)) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (!aligned_to(mismatches, 8)) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  return launch_lds_atomic_order_selftest(static_cast<hipStream_t>(stream), rows,
                                          mismatches);
}

int32_t ilgpu_hip_radix_sort_passes(ilgpu_hip_stream_t stream, const void* temp,
                                    int64_t temp_bytes, int64_t n, int32_t key_type,
                                    int32_t value_bytes, int32_t* executed,
                                    int32_t* skipped) {
  if (executed == nullptr || skipped == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  const int kb = elem_size(key_type);
  if (kb < 0) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (value_bytes != 0 && value_bytes != 1 && value_bytes != 2 && value_bytes != 4 &&
      value_bytes != 8 && value_bytes != 16)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (n < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (n > radix_sort_max_length()) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  const int32_t rc = check_temp(temp, temp_bytes, radix_sort_temp_bytes(n, kb, value_bytes));
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  return read_sort_plan(static_cast<hipStream_t>(stream), temp, n, kb, value_bytes, executed,
                        skipped);
}

int32_t ilgpu_hip_sort_check_device(ilgpu_hip_stream_t stream) {
  return check_sort_device(static_cast<hipStream_t>(stream));
}

int32_t ilgpu_hip_sort_set_parameter(int32_t parameter, int32_t value) {
  if (parameter != ILGPU_HIP_SORT_PARAM_LOOKBACK_SPIN_LIMIT &&
      parameter != ILGPU_HIP_SORT_PARAM_LARGE_BLOCK_MIN_TILES_PER_CU &&
      parameter != ILGPU_HIP_SORT_PARAM_ONE_TILE_KERNEL &&
      parameter != ILGPU_HIP_SORT_PARAM_ASSUME_LDS_ATOMIC_ORDER &&
      parameter != ILGPU_HIP_SORT_PARAM_SHORT_TILE_MAX_TILES)
    return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  set_sort_parameter(parameter, value);
  return ILGPU_HIP_SUCCESS;
}

/* ---- scan -------------------------------------------------------------- */

int32_t ilgpu_hip_scan_temp_bytes(int64_t n, int32_t elem_type,
                                  int64_t* temp_bytes) {
  if (temp_bytes == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (!scan_reduce_type(elem_type)) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (n < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (n > INT32_MAX) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  *temp_bytes = scan_temp_bytes(n, elem_size(elem_type));
  return ILGPU_HIP_SUCCESS;
}

int32_t ilgpu_hip_scan(ilgpu_hip_stream_t stream, const void* in,
                       int64_t in_length, int64_t in_stride, void* out,
                       int64_t out_length, int64_t out_stride,
                       int32_t elem_type, int32_t op, int32_t kind, void* temp,
                       int64_t temp_bytes) {
  /* Order of checks as in ScanExtensions.cs:675-685. */
  if (!scan_reduce_type(elem_type) || !valid_op(op) ||
      (kind != ILGPU_HIP_SCAN_INCLUSIVE && kind != ILGPU_HIP_SCAN_EXCLUSIVE))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!valid_view(in, in_length)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (!valid_view(out, out_length)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (out_length < in_length) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (in_length > INT32_MAX) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  const int eb = elem_size(elem_type);
  if (in_stride < 1 || out_stride < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (!aligned_to(in, eb) || !aligned_to(out, eb))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  const int32_t rc = check_temp(temp, temp_bytes, scan_temp_bytes(in_length, eb));
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  return launch_scan(static_cast<hipStream_t>(stream), in, in_stride, out,
                     out_stride, in_length, elem_type, op, kind, temp);
}

int32_t ilgpu_hip_scan_static(ilgpu_hip_stream_t stream, const void* in,
                              int64_t in_length, int64_t in_stride, void* out,
                              int64_t out_length, int64_t out_stride,
                              int32_t elem_type, int32_t op, int32_t kind) {
  /* The checks of ilgpu_hip_scan, in its order; no temp to check. */
  if (!scan_reduce_type(elem_type) || !valid_op(op) ||
      (kind != ILGPU_HIP_SCAN_INCLUSIVE && kind != ILGPU_HIP_SCAN_EXCLUSIVE))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!valid_view(in, in_length)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (!valid_view(out, out_length)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (out_length < in_length) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (in_length > INT32_MAX) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  const int eb = elem_size(elem_type);
  if (in_stride < 1 || out_stride < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (!aligned_to(in, eb) || !aligned_to(out, eb))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (in_length * eb > ILGPU_HIP_SCAN_STATIC_MAX_BYTES)
    return ILGPU_HIP_ERROR_STATIC_LIMIT;
  return launch_scan_static(static_cast<hipStream_t>(stream), in, in_stride, out,
                            out_stride, in_length, elem_type, op, kind);
}

/* ---- reduce ------------------------------------------------------------ */

int32_t ilgpu_hip_reduce_temp_bytes(int64_t n, int32_t elem_type,
                                    int64_t* temp_bytes) {
  if (temp_bytes == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (!scan_reduce_type(elem_type)) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (n < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  *temp_bytes = reduce_temp_bytes();
  return ILGPU_HIP_SUCCESS;
}

int32_t ilgpu_hip_reduce(ilgpu_hip_stream_t stream, const void* in, int64_t n,
                         int64_t stride, int32_t elem_type, int32_t op,
                         void* out, int64_t out_length, void* temp,
                         int64_t temp_bytes) {
  /* Order of checks as in ReductionExtensions.cs:146-153. */
  if (!scan_reduce_type(elem_type) || !valid_op(op))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!valid_view(in, n)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (!valid_view(out, out_length)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (n > INT32_MAX) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  const int eb = elem_size(elem_type);
  if (stride < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (!aligned_to(in, eb) || !aligned_to(out, eb))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  const int32_t rc = check_temp(temp, temp_bytes, reduce_temp_bytes());
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  return launch_reduce(static_cast<hipStream_t>(stream), in, n, stride,
                       elem_type, op, out, temp);
}

/* ---- histogram --------------------------------------------------------- */

int32_t ilgpu_hip_histogram(ilgpu_hip_stream_t stream, const void* in,
                            int64_t n, int64_t stride, int32_t in_type,
                            void* bins, int64_t num_bins, int32_t bin_type,
                            int32_t locator, int32_t* overflow) {
  /* Order of checks as in HistogramExtensions.cs:322-338. */
  const int eb = elem_size(in_type);
  if (eb < 0 || in_type == ILGPU_HIP_F16) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (bin_type != ILGPU_HIP_I32 && bin_type != ILGPU_HIP_U32 &&
      bin_type != ILGPU_HIP_I64 && bin_type != ILGPU_HIP_U64 &&
      bin_type != ILGPU_HIP_F32 && bin_type != ILGPU_HIP_F64)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (locator != ILGPU_HIP_LOCATOR_IDENTITY &&
      locator != ILGPU_HIP_LOCATOR_MODULO)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!valid_view(in, n)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (!valid_view(bins, num_bins)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (n > INT32_MAX || num_bins > INT32_MAX) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (stride < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (!aligned_to(in, eb) || !aligned_to(bins, elem_size(bin_type)) ||
      (overflow != nullptr && !aligned_to(overflow, 4)))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  return launch_histogram(static_cast<hipStream_t>(stream), in, n, stride,
                          in_type, bins, num_bins, bin_type, locator, overflow);
}

/* ---- unique ------------------------------------------------------------ */

int32_t ilgpu_hip_unique_temp_bytes(int64_t n, int32_t elem_type,
                                    int64_t* temp_bytes) {
  if (temp_bytes == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  const int eb = elem_size(elem_type);
  if (eb < 0) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (n < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (n > INT32_MAX) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  *temp_bytes = unique_temp_bytes(n, eb);
  return ILGPU_HIP_SUCCESS;
}

int32_t ilgpu_hip_unique(ilgpu_hip_stream_t stream, void* input, int64_t n,
                         int32_t elem_type, int64_t* new_length,
                         int64_t new_length_extent, void* temp,
                         int64_t temp_bytes) {
  /* Order of checks as in UniqueExtensions.cs:160-178. */
  const int eb = elem_size(elem_type);
  if (eb < 0) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!valid_view(input, n)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (!valid_view(new_length, new_length_extent)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (temp == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (n > INT32_MAX) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!aligned_to(input, eb) || !aligned_to(new_length, 8))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  const int32_t rc = check_temp(temp, temp_bytes, unique_temp_bytes(n, eb));
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  return launch_unique(static_cast<hipStream_t>(stream), input, n, elem_type,
                       new_length, temp);
}

/* ---- initialize, sequence, reorder -------------------------------------- */

int32_t ilgpu_hip_initialize(ilgpu_hip_stream_t stream, void* view, int64_t n,
                             int64_t stride, int32_t elem_bytes,
                             const void* value) {
  /* InitializeExtensions.cs:124-127. */
  if (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4 &&
      elem_bytes != 8 && elem_bytes != 16)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!valid_view(view, n) || value == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (stride < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (!aligned_to(view, elem_bytes)) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  return launch_initialize(static_cast<hipStream_t>(stream), view, n, stride,
                           elem_bytes, value);
}

int32_t ilgpu_hip_sequence(ilgpu_hip_stream_t stream, void* view, int64_t n,
                           int64_t stride, int32_t elem_type,
                           int64_t sequence_length, int64_t batch_length) {
  /* SequenceExtensions.cs:362-371. */
  const int eb = elem_size(elem_type);
  if (eb < 0) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!valid_view(view, n)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (sequence_length < 1 || batch_length < 1 || stride < 1)
    return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (!aligned_to(view, eb)) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  return launch_sequence(static_cast<hipStream_t>(stream), view, n, stride,
                         elem_type, sequence_length, batch_length);
}

int32_t ilgpu_hip_reorder(ilgpu_hip_stream_t stream, const void* source,
                          int64_t source_length, void* target,
                          int64_t target_length, const int32_t* order,
                          int64_t order_length, int32_t elem_bytes) {
  /* ReorderExtensions.cs:158-171, then TransformExtensions.cs:318-332 with the
   * order view as the transformer's source. */
  if (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4 &&
      elem_bytes != 8 && elem_bytes != 16)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!valid_view(source, source_length)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (!valid_view(order, order_length)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (order_length < source_length) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (source_length > INT32_MAX) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!valid_view(target, target_length)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (target_length < order_length) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (!aligned_to(source, elem_bytes) || !aligned_to(target, elem_bytes) ||
      !aligned_to(order, 4))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  return launch_reorder(static_cast<hipStream_t>(stream), source, target, order,
                        order_length, elem_bytes);
}

/* ---- transform, reorder-transform --------------------------------------- */

static int32_t check_transformer(int32_t source_type, int32_t target_type,
                                 int32_t transformer) {
  if (elem_size(source_type) < 0 || elem_size(target_type) < 0)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (transformer < ILGPU_HIP_TRANSFORM_CONVERT ||
      transformer > ILGPU_HIP_TRANSFORM_MULTIPLY)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  const bool float_source = source_type >= ILGPU_HIP_F16;
  const bool float_target = target_type >= ILGPU_HIP_F16;
  if (float_source && !float_target) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (float_source && transformer == ILGPU_HIP_TRANSFORM_BIT_COMPLEMENT)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  return ILGPU_HIP_SUCCESS;
}

int32_t ilgpu_hip_transform(ilgpu_hip_stream_t stream, const void* source,
                            int64_t source_length, int64_t source_stride,
                            int32_t source_type, void* target,
                            int64_t target_length, int64_t target_stride,
                            int32_t target_type, int32_t transformer,
                            int64_t factor) {
  /* TransformExtensions.cs:304-317. */
  const int32_t rc = check_transformer(source_type, target_type, transformer);
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  if (!valid_view(source, source_length)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (target == nullptr || target_length < 0) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (target_length < source_length) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (source_stride < 1 || target_stride < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (!aligned_to(source, elem_size(source_type)) ||
      !aligned_to(target, elem_size(target_type)))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  TransformArgs a{source, source_stride, source_type, target, target_stride,
                  target_type, nullptr, source_length, transformer, factor};
  return launch_transform(static_cast<hipStream_t>(stream), a);
}

int32_t ilgpu_hip_reorder_transform(ilgpu_hip_stream_t stream,
                                    const void* source, int64_t source_length,
                                    int32_t source_type, void* target,
                                    int64_t target_length, int32_t target_type,
                                    const int32_t* order, int64_t order_length,
                                    int32_t transformer, int64_t factor) {
  /* ReorderExtensions.cs:158-171, then TransformExtensions.cs:304-317 with
   * the order view as the transformer's source. */
  const int32_t rc = check_transformer(source_type, target_type, transformer);
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  if (!valid_view(source, source_length)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (!valid_view(order, order_length)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (order_length < source_length) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (source_length > INT32_MAX) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!valid_view(target, target_length)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (target_length < order_length) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (!aligned_to(source, elem_size(source_type)) ||
      !aligned_to(target, elem_size(target_type)) || !aligned_to(order, 4))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  TransformArgs a{source, 1, source_type, target, 1, target_type, order,
                  order_length, transformer, factor};
  return launch_transform(static_cast<hipStream_t>(stream), a);
}

/* ---- embedding ----------------------------------------------------------- */

static int32_t check_tokens(const void* tokens, int64_t count, int32_t token_type) {
  if (token_type != ILGPU_HIP_I32 && token_type != ILGPU_HIP_I64)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (count < 0) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (count > INT32_MAX) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (count > 0 && tokens == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (!aligned_to(tokens, elem_size(token_type))) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  return ILGPU_HIP_SUCCESS;
}

int32_t ilgpu_hip_embedding(ilgpu_hip_stream_t stream, const void* table,
                            int64_t vocabulary, int64_t dimension,
                            int64_t table_stride, int32_t table_type,
                            const void* tokens, int64_t count,
                            int32_t token_type, const float* scale, void* out,
                            int64_t out_stride, int32_t out_type) {
  const int tb = operator_elem_size(table_type), ob = operator_elem_size(out_type);
  if (tb < 0 || ob < 0) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  int32_t rc = check_tokens(tokens, count, token_type);
  if (rc == ILGPU_HIP_SUCCESS)
    rc = check_matrix(table, vocabulary, dimension, table_stride, tb, false);
  if (rc == ILGPU_HIP_SUCCESS) rc = check_matrix(out, count, dimension, out_stride, ob, true);
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  const EmbeddingArgs a{table, vocabulary, dimension, table_stride, table_type, tokens, count,
                        token_type, scale != nullptr ? *scale : 1.0f, out, out_stride, out_type};
  return launch_embedding(static_cast<hipStream_t>(stream), a);
}

int32_t ilgpu_hip_embedding_gradient_temp_bytes(int64_t count, int64_t vocabulary,
                                                int64_t dimension, int64_t* temp_bytes) {
  if (temp_bytes == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (count < 0 || vocabulary < 0 || dimension < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (count > radix_sort_max_length() || vocabulary > INT32_MAX || dimension > INT32_MAX)
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  *temp_bytes = embedding_gradient_temp_bytes(count, vocabulary, dimension);
  return ILGPU_HIP_SUCCESS;
}

int32_t ilgpu_hip_embedding_gradient(
    ilgpu_hip_stream_t stream, const void* grad_out, int64_t grad_out_stride,
    int32_t grad_out_type, const void* tokens, int64_t count,
    int32_t token_type, const float* scale, int64_t padding_token,
    int32_t accumulate, void* grad_table, int64_t vocabulary,
    int64_t dimension, int64_t grad_table_stride, int32_t grad_table_type,
    void* temp, int64_t temp_bytes) {
  const int gb = operator_elem_size(grad_out_type), wb = operator_elem_size(grad_table_type);
  if (gb < 0 || wb < 0) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  int32_t rc = check_tokens(tokens, count, token_type);
  if (rc == ILGPU_HIP_SUCCESS && count > radix_sort_max_length())
    rc = ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (rc == ILGPU_HIP_SUCCESS)
    rc = check_matrix(grad_out, count, dimension, grad_out_stride, gb, false);
  if (rc == ILGPU_HIP_SUCCESS)
    rc = check_matrix(grad_table, vocabulary, dimension, grad_table_stride, wb, true);
  if (rc == ILGPU_HIP_SUCCESS)
    rc = check_temp(temp, temp_bytes, embedding_gradient_temp_bytes(count, vocabulary, dimension));
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  const EmbeddingGradientArgs a{grad_out, grad_out_stride, grad_out_type, tokens, count,
                                token_type, scale != nullptr ? *scale : 1.0f, padding_token,
                                accumulate != 0 ? 1 : 0, grad_table, vocabulary, dimension,
                                grad_table_stride, grad_table_type, temp};
  return launch_embedding_gradient(static_cast<hipStream_t>(stream), a);
}

/* ---- layer norm ------------------------------------------------------------ */

static int32_t check_norm_types(int32_t type, int32_t weight_type) {
  if (operator_elem_size(type) < 0 || (weight_type != type && weight_type != ILGPU_HIP_F32))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  return ILGPU_HIP_SUCCESS;
}

int32_t ilgpu_hip_layer_norm(ilgpu_hip_stream_t stream, const void* in,
                             int64_t rows, int64_t columns, int64_t in_stride,
                             int32_t type, const void* weight,
                             const void* bias, int32_t weight_type,
                             const float* epsilon, void* out,
                             int64_t out_stride, float* mean, float* rstd) {
  int32_t rc = check_norm_types(type, weight_type);
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  const int eb = operator_elem_size(type), wb = operator_elem_size(weight_type);
  if (epsilon == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  rc = check_matrix(in, rows, columns, in_stride, eb, false);
  if (rc == ILGPU_HIP_SUCCESS) rc = check_matrix(out, rows, columns, out_stride, eb, true);
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  if (!(*epsilon >= 0.0f && *epsilon <= 3.402823466e+38f)) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (!aligned_to(weight, wb) || !aligned_to(bias, wb) || !aligned_to(mean, 4) ||
      !aligned_to(rstd, 4))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  const LayerNormArgs a{in, rows, columns, in_stride, type, weight, bias, weight_type,
                        *epsilon, out, out_stride, mean, rstd};
  return launch_layer_norm(static_cast<hipStream_t>(stream), a);
}

int32_t ilgpu_hip_layer_norm_gradient_temp_bytes(int64_t rows, int64_t columns,
                                                 int64_t* temp_bytes) {
  if (temp_bytes == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (rows < 0 || columns < 1) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (rows > INT32_MAX || columns > INT32_MAX) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  *temp_bytes = layer_norm_gradient_temp_bytes(rows, columns);
  return ILGPU_HIP_SUCCESS;
}

int32_t ilgpu_hip_layer_norm_gradient(
    ilgpu_hip_stream_t stream, const void* grad_out, int64_t grad_out_stride,
    const void* in, int64_t in_stride, int64_t rows, int64_t columns,
    int32_t type, const void* weight, int32_t weight_type, const float* mean,
    const float* rstd, void* grad_in, int64_t grad_in_stride,
    void* grad_weight, void* grad_bias, int32_t accumulate, void* temp,
    int64_t temp_bytes) {
  int32_t rc = check_norm_types(type, weight_type);
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  const int eb = operator_elem_size(type), wb = operator_elem_size(weight_type);
  rc = check_matrix(grad_out, rows, columns, grad_out_stride, eb, false);
  if (rc == ILGPU_HIP_SUCCESS) rc = check_matrix(in, rows, columns, in_stride, eb, false);
  if (rc == ILGPU_HIP_SUCCESS && grad_in != nullptr)
    rc = check_matrix(grad_in, rows, columns, grad_in_stride, eb, true);
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  if (rows > 0 && (mean == nullptr || rstd == nullptr)) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (rows > 0 && grad_in == nullptr && grad_weight == nullptr && grad_bias == nullptr)
    return ILGPU_HIP_ERROR_NULL_VIEW;
  if (!aligned_to(weight, wb) || !aligned_to(grad_weight, wb) || !aligned_to(grad_bias, wb) ||
      !aligned_to(mean, 4) || !aligned_to(rstd, 4))
    return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  rc = check_temp(temp, temp_bytes, layer_norm_gradient_temp_bytes(rows, columns));
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  const LayerNormGradientArgs a{grad_out, grad_out_stride, in, in_stride, rows, columns, type,
                                weight, weight_type, mean, rstd, grad_in, grad_in_stride,
                                grad_weight, grad_bias, accumulate != 0 ? 1 : 0, temp};
  return launch_layer_norm_gradient(static_cast<hipStream_t>(stream), a);
}

/* ---- gradient norm and clipping ---------------------------------------------- */

int32_t ilgpu_hip_gradient_norm_temp_bytes(int64_t count, int64_t* temp_bytes) {
  if (temp_bytes == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (count < 0) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  if (count > INT32_MAX) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  *temp_bytes = gradient_norm_temp_bytes(count);
  return ILGPU_HIP_SUCCESS;
}

int32_t ilgpu_hip_gradient_norm(ilgpu_hip_stream_t stream,
                                const ilgpu_hip_tensor* tensors, int64_t count,
                                float* norm, void* temp, int64_t temp_bytes) {
  int32_t rc = check_tensors(tensors, count);
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  if (norm == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (!aligned_to(norm, 4)) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  rc = check_temp(temp, temp_bytes, gradient_norm_temp_bytes(count));
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  return launch_gradient_norm(static_cast<hipStream_t>(stream), tensors, count, norm, temp);
}

int32_t ilgpu_hip_clip_gradients(ilgpu_hip_stream_t stream,
                                 const ilgpu_hip_tensor* sources,
                                 const ilgpu_hip_tensor* targets, int64_t count,
                                 const float* norm, const float* max_norm) {
  int32_t rc = check_tensors(sources, count);
  if (rc == ILGPU_HIP_SUCCESS && targets != nullptr) rc = check_tensors(targets, count);
  if (rc != ILGPU_HIP_SUCCESS) return rc;
  for (int64_t k = 0; targets != nullptr && k < count; ++k) {
    if (targets[k].type != sources[k].type) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
    if (targets[k].length != sources[k].length) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  }
  if (norm == nullptr || max_norm == nullptr) return ILGPU_HIP_ERROR_NULL_VIEW;
  if (!aligned_to(norm, 4)) return ILGPU_HIP_ERROR_NOT_SUPPORTED;
  if (!(*max_norm >= 0.0f)) return ILGPU_HIP_ERROR_OUT_OF_RANGE;
  return launch_clip_gradients(static_cast<hipStream_t>(stream), sources, targets, count, norm,
                               *max_norm);
}

}  // extern "C"
