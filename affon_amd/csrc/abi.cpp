// C ABI of the rocm quantized-linear backend: sessions, device memory,
// validation, implementation selection and the host-pointer drop-in.
//
// Validation mirrors the reference exactly:
//   src/js/compute/program.ts:481-494      (operand dtypes, bits, group, shapes)
//   src/support/compute_core_cyna.zig:1000-1022 (overflow-checked counts)
// and rejects before any device work, leaving the output untouched.

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <exception>
#include <initializer_list>
#include <limits>
#include <memory>
#include <mutex>
#include <string>
#include <vector>

#include "affon_rocm.h"
#include "internal.h"
#include "overlap.h"

struct affon_rocm_session {
  int device = 0;
  hipStream_t stream = nullptr;
  affon::Workspace* workspace = nullptr;
  // Allocations made through affon_rocm_alloc; the session frees those still
  // live when it ends, so tensors that outlive it leak nothing.
  affon::DeviceMemory* memory = nullptr;
};

// Scratch memory of affon_rocm_quantized_matmul_noalloc: the split-K partial
// sums of the tiled kernels and the reassociated prefill GEMM's per-group
// activation sums, in a static device array (one per GPU, held until the
// process ends): 32 MiB of partial sums (four K ranges of a 512 x 4096 f32
// output) plus 1 MiB of group sums. Host code uses only the per-device
// address that hipGetSymbolAddress returns for it (kept by scratch_on), never
// the array's name, which on the host is a stand-in and not a device address.
constexpr size_t kNoAllocScratchBytes = (size_t(32) << 20) + (size_t(1) << 20);
static __device__ __align__(256) uint8_t scratch[kNoAllocScratchBytes];

namespace {

// Device address of `scratch` on `device`, looked up on the first
// no-allocation call on that device, with the device current (check_session
// has made it so); only a successful lookup is kept, so a failed one is
// retried by the next call.
std::mutex g_scratch_mutex;
void* g_scratch_ptr[64] = {};

hipError_t scratch_on(int device, void** out) {
  *out = nullptr;
  if (device < 0 || device >= 64) return hipErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(g_scratch_mutex);
  if (g_scratch_ptr[device] == nullptr) {
    void* ptr = nullptr;
    const hipError_t e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));
    if (e != hipSuccess) return e;
    g_scratch_ptr[device] = ptr;
  }
  *out = g_scratch_ptr[device];
  return hipSuccess;
}

thread_local std::string g_last_error;

int fail(int status, const char* format, ...) {
  char buffer[512];
  va_list args;
  va_start(args, format);
  std::vsnprintf(buffer, sizeof(buffer), format, args);
  va_end(args);
  g_last_error = buffer;
  return status;
}

int hip_fail(hipError_t error, const char* what) {
  return fail(AFFON_ROCM_HIP_ERROR, "%s: %s", what, hipGetErrorString(error));
}

// Of a launch that does nothing without the session's workspace.
int workspace_fail(hipError_t error, const char* what) {
  if (error != hipErrorOutOfMemory) return hip_fail(error, what);
  return fail(AFFON_ROCM_HIP_ERROR,
              "%s needs a larger workspace, which there is no memory for, or which a stream that is captured cannot get: run "
              "the call once before the capture", what);
}

void clear_error() { g_last_error.clear(); }

bool mul_ok(uint64_t a, uint64_t b, uint64_t* out) {
  if (a != 0 && b > std::numeric_limits<uint64_t>::max() / a) return false;
  *out = a * b;
  return true;
}

bool add_ok(uint64_t a, uint64_t b, uint64_t* out) {
  if (b > std::numeric_limits<uint64_t>::max() - a) return false;
  *out = a + b;
  return true;
}

int element_size(int dtype) {
  switch (dtype) {
    case AFFON_ROCM_F32: return 4;
    case AFFON_ROCM_BF16: return 2;
    case AFFON_ROCM_U32: return 4;
    default: return 0;
  }
}

bool is_float_dtype(int dtype) { return dtype == AFFON_ROCM_F32 || dtype == AFFON_ROCM_BF16; }

// Checks that every element a view names lies inside its allocation.
int check_view(const affon_rocm_view& v, const char* name, const char* op = "quantized_matmul") {
  const int esize = element_size(v.dtype);
  if (v.data == nullptr) return fail(AFFON_ROCM_INVALID_SHAPE, "%s %s has no data", op, name);
  if (v.shape[0] <= 0 || v.shape[1] <= 0)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s %s has an empty dimension", op, name);
  if (v.stride[0] < 0 || v.stride[1] < 0)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s %s has a negative stride", op, name);
  if (v.byte_offset % static_cast<size_t>(esize) != 0)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s %s byte offset is not element aligned", op, name);
  uint64_t last0 = 0, last1 = 0, last = 0, bytes = 0, end = 0;
  if (!mul_ok(static_cast<uint64_t>(v.shape[0] - 1), static_cast<uint64_t>(v.stride[0]), &last0) ||
      !mul_ok(static_cast<uint64_t>(v.shape[1] - 1), static_cast<uint64_t>(v.stride[1]), &last1) ||
      !add_ok(last0, last1, &last) || !add_ok(last, 1, &last) ||
      !mul_ok(last, static_cast<uint64_t>(esize), &bytes) ||
      !add_ok(bytes, static_cast<uint64_t>(v.byte_offset), &end))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s %s extent overflows", op, name);
  if (end > v.buffer_bytes)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s %s view exceeds its buffer (%llu > %llu bytes)", op, name,
                static_cast<unsigned long long>(end), static_cast<unsigned long long>(v.buffer_bytes));
  return AFFON_ROCM_OK;
}

// program.ts:483-493 and compute_core_cyna.zig:1012-1022.
int validate(const affon_rocm_qmm_desc* d, affon::QmmProblem* p) {
  if (d == nullptr) return fail(AFFON_ROCM_INVALID_SHAPE, "quantized_matmul descriptor is null");
  if (d->bits != 2 && d->bits != 4 && d->bits != 8)
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantized_matmul bits must be 2, 4, or 8");
  if (d->group_size == 0)
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantized_matmul group_size must be a positive integer");
  if (!is_float_dtype(d->input.dtype) || d->packed.dtype != AFFON_ROCM_U32 || !is_float_dtype(d->scales.dtype) ||
      d->biases.dtype != d->scales.dtype)
    return fail(AFFON_ROCM_INVALID_SHAPE,
                "quantized_matmul requires f32/bf16 input, u32 weights, and matching f32/bf16 scales and biases");
  const int64_t M = d->input.shape[0], K = d->input.shape[1], N = d->packed.shape[0];
  const int64_t per_word = 32 / static_cast<int64_t>(d->bits);
  const int64_t g = static_cast<int64_t>(d->group_size);
  if (M <= 0 || K <= 0 || N <= 0 || K % per_word != 0 || K % g != 0 || d->packed.shape[1] != K / per_word ||
      d->scales.shape[0] != N || d->scales.shape[1] != K / g || d->biases.shape[0] != N ||
      d->biases.shape[1] != K / g)
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantized_matmul packed or group dimensions do not match input features");
  int status;
  if ((status = check_view(d->input, "input")) != AFFON_ROCM_OK) return status;
  if ((status = check_view(d->packed, "packed")) != AFFON_ROCM_OK) return status;
  if ((status = check_view(d->scales, "scales")) != AFFON_ROCM_OK) return status;
  if ((status = check_view(d->biases, "biases")) != AFFON_ROCM_OK) return status;
  uint64_t out_count = 0, out_bytes = 0;
  if (!mul_ok(static_cast<uint64_t>(M), static_cast<uint64_t>(N), &out_count) || !mul_ok(out_count, 4, &out_bytes))
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantized_matmul output size overflows");
  if (d->output == nullptr || d->output_bytes < out_bytes)
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantized_matmul output buffer is smaller than [M,N] f32");
  if (d->implementation < AFFON_ROCM_IMPL_AUTO || d->implementation > AFFON_ROCM_IMPL_MFMA)
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantized_matmul unknown implementation %d", d->implementation);
  if (d->numerical_policy < AFFON_ROCM_BACKEND_EQUIVALENT || d->numerical_policy > AFFON_ROCM_APPROXIMATE)
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantized_matmul unknown numerical policy %d", d->numerical_policy);

  p->M = M;
  p->N = N;
  p->K = K;
  p->bits = static_cast<int>(d->bits);
  p->group = g;
  p->x = static_cast<const uint8_t*>(d->input.data) + d->input.byte_offset;
  p->xs0 = d->input.stride[0];
  p->xs1 = d->input.stride[1];
  p->x_dtype = d->input.dtype;
  p->w = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(d->packed.data) + d->packed.byte_offset);
  p->ws0 = d->packed.stride[0];
  p->ws1 = d->packed.stride[1];
  p->s = static_cast<const uint8_t*>(d->scales.data) + d->scales.byte_offset;
  p->ss0 = d->scales.stride[0];
  p->ss1 = d->scales.stride[1];
  p->b = static_cast<const uint8_t*>(d->biases.data) + d->biases.byte_offset;
  p->bs0 = d->biases.stride[0];
  p->bs1 = d->biases.stride[1];
  p->p_dtype = d->scales.dtype;
  p->out = d->output;
  return AFFON_ROCM_OK;
}

// Registered candidates, in the order AUTO prefers them.
struct Candidate {
  int impl;
  const char* id;
  int version;
  // 0 exact (bit-identical to the ordered CPU loop), 1 reassociated,
  // 2 approximate (rounds decoded weights to bf16).
  int numerical_class;
  bool (*supports)(const affon::QmmProblem&);
  hipError_t (*launch)(const affon::QmmProblem&, const affon::Launch&);
};

const Candidate kCandidates[] = {
    {AFFON_ROCM_IMPL_MFMA, "rocm_quantized_matmul.mfma", 1, 2, affon::mfma_supports, affon::mfma_launch},
    {AFFON_ROCM_IMPL_GEMV_MFMA, "rocm_quantized_matmul.gemv_mfma", 1, 1, affon::gemv_mfma_supports,
     affon::gemv_mfma_launch},
    {AFFON_ROCM_IMPL_GEMV, "rocm_quantized_matmul.gemv", 1, 1, affon::gemv_supports, affon::gemv_launch},
    {AFFON_ROCM_IMPL_GENERIC, "rocm_quantized_matmul.generic", 1, 0, affon::generic_supports,
     affon::generic_launch},
};

bool policy_accepts(int policy, int numerical_class) {
  switch (policy) {
    case AFFON_ROCM_EXACT_ONLY: return numerical_class == 0;
    case AFFON_ROCM_BACKEND_EQUIVALENT: return numerical_class <= 1;
    default: return true;
  }
}

// Shape rule for AUTO among candidates that pass their guards: the prefill
// GEMM for M >= 64 (when the policy admits its approximate class), the MFMA
// decode kernels for M >= 2 with bf16 input (the reassociated class's path
// for prefill: from 128 rows the large-tile reassociated GEMM, gemm_re.hip,
// where it takes the shape, else row tiles of 32), otherwise the gemv candidate
// (one row, f32 activations, and the layouts those decline), the generic
// kernel last.
bool auto_prefers(const Candidate& c, const affon::QmmProblem& p) {
  switch (c.impl) {
    case AFFON_ROCM_IMPL_MFMA: return p.M >= 64;
    case AFFON_ROCM_IMPL_GEMV_MFMA: return p.M >= 2;
    default: return true;
  }
}

int select(const affon_rocm_qmm_desc* d, const affon::QmmProblem& p, const Candidate** out) {
  for (const Candidate& c : kCandidates) {
    if (d->implementation != AFFON_ROCM_IMPL_AUTO && d->implementation != c.impl) continue;
    if (!policy_accepts(d->numerical_policy, c.numerical_class)) {
      if (d->implementation == c.impl)
        return fail(AFFON_ROCM_UNSUPPORTED, "%s is not allowed under the requested numerical policy", c.id);
      continue;
    }
    if (!c.supports(p)) {
      if (d->implementation == c.impl)
        return fail(AFFON_ROCM_UNSUPPORTED, "%s cannot run this shape or layout", c.id);
      continue;
    }
    if (d->implementation == AFFON_ROCM_IMPL_AUTO && !auto_prefers(c, p)) continue;
    *out = &c;
    return AFFON_ROCM_OK;
  }
  return fail(AFFON_ROCM_UNSUPPORTED, "no quantized_matmul implementation accepts this problem");
}

int check_session(affon_rocm_session* s) {
  if (s == nullptr || s->stream == nullptr) return fail(AFFON_ROCM_CORE_FAILURE, "session is not open");
  hipError_t e = hipSetDevice(s->device);
  if (e != hipSuccess) return hip_fail(e, "hipSetDevice");
  return AFFON_ROCM_OK;
}

bool is_gfx950(int device) {
  hipDeviceProp_t prop;
  if (hipGetDeviceProperties(&prop, device) != hipSuccess) return false;
  return std::strncmp(prop.gcnArchName, "gfx950", 6) == 0;
}

}  // namespace

extern "C" {

int affon_rocm_device_count(int* count) {
  clear_error();
  if (count == nullptr) return fail(AFFON_ROCM_CORE_FAILURE, "count is null");
  *count = 0;
  int n = 0;
  hipError_t e = hipGetDeviceCount(&n);
  if (e == hipErrorNoDevice) return AFFON_ROCM_OK;
  if (e != hipSuccess) return hip_fail(e, "hipGetDeviceCount");
  for (int i = 0; i < n; ++i) *count += is_gfx950(i) ? 1 : 0;
  return AFFON_ROCM_OK;
}

int affon_rocm_session_create(int device, affon_rocm_session** out) {
  clear_error();
  if (out == nullptr) return fail(AFFON_ROCM_CORE_FAILURE, "session output is null");
  int n = 0;
  hipError_t e = hipGetDeviceCount(&n);
  if (e != hipSuccess || device < 0 || device >= n)
    return fail(AFFON_ROCM_UNSUPPORTED, "rocm backend unavailable: no HIP device %d", device);
  if (!is_gfx950(device)) return fail(AFFON_ROCM_UNSUPPORTED, "rocm backend unavailable: device %d is not gfx950", device);
  if ((e = hipSetDevice(device)) != hipSuccess) return hip_fail(e, "hipSetDevice");
  hipStream_t stream = nullptr;
  if ((e = hipStreamCreateWithFlags(&stream, hipStreamNonBlocking)) != hipSuccess) return hip_fail(e, "hipStreamCreate");
  try {
    auto workspace = std::make_unique<affon::Workspace>(device, stream);
    auto memory = std::make_unique<affon::DeviceMemory>(stream);
    *out = new affon_rocm_session{device, stream, workspace.get(), memory.get()};
    workspace.release();
    memory.release();
  } catch (const std::exception& error) {
    (void)hipStreamDestroy(stream);
    return fail(AFFON_ROCM_CORE_FAILURE, "session_create: %s", error.what());
  }
  return AFFON_ROCM_OK;
}

int affon_rocm_session_destroy(affon_rocm_session* session) {
  clear_error();
  if (session == nullptr) return AFFON_ROCM_OK;
  int status = AFFON_ROCM_OK;
  if (hipSetDevice(session->device) == hipSuccess && session->stream != nullptr) {
    hipError_t e = hipStreamSynchronize(session->stream);
    if (e != hipSuccess) status = hip_fail(e, "hipStreamSynchronize");
    session->memory->release_all();
    delete session->workspace;
    e = hipStreamDestroy(session->stream);
    if (e != hipSuccess && status == AFFON_ROCM_OK) status = hip_fail(e, "hipStreamDestroy");
  } else {
    delete session->workspace;
  }
  delete session->memory;
  delete session;
  return status;
}

void* affon_rocm_session_stream(affon_rocm_session* session) {
  return session == nullptr ? nullptr : static_cast<void*>(session->stream);
}

int affon_rocm_alloc(affon_rocm_session* session, size_t bytes, void** out) {
  clear_error();
  int status = check_session(session);
  if (status != AFFON_ROCM_OK) return status;
  if (out == nullptr) return fail(AFFON_ROCM_CORE_FAILURE, "allocation output is null");
  *out = nullptr;
  try {
    const hipError_t e = session->memory->alloc(bytes, out);
    if (e != hipSuccess) return hip_fail(e, "hipMalloc");
  } catch (const std::exception& e) {
    return fail(AFFON_ROCM_CORE_FAILURE, "alloc: %s", e.what());
  }
  return AFFON_ROCM_OK;
}

int affon_rocm_free(affon_rocm_session* session, void* ptr) {
  clear_error();
  int status = check_session(session);
  if (status != AFFON_ROCM_OK) return status;
  if (ptr == nullptr) return AFFON_ROCM_OK;
  hipError_t e = hipSuccess;
  try {
    if (!session->memory->free(ptr, &e))
      return fail(AFFON_ROCM_CORE_FAILURE, "free of memory this session did not allocate");
  } catch (const std::exception& error) {
    return fail(AFFON_ROCM_CORE_FAILURE, "free: %s", error.what());
  }
  if (e != hipSuccess) return hip_fail(e, "hipFree");
  return AFFON_ROCM_OK;
}

static int copy(affon_rocm_session* session, void* dst, const void* src, size_t bytes, hipMemcpyKind kind) {
  clear_error();
  int status = check_session(session);
  if (status != AFFON_ROCM_OK) return status;
  if (bytes == 0) return AFFON_ROCM_OK;
  if (dst == nullptr || src == nullptr) return fail(AFFON_ROCM_CORE_FAILURE, "copy with a null pointer");
  hipError_t e = hipMemcpyAsync(dst, src, bytes, kind, session->stream);
  if (e != hipSuccess) return hip_fail(e, "hipMemcpyAsync");
  e = hipStreamSynchronize(session->stream);
  if (e != hipSuccess) return hip_fail(e, "hipStreamSynchronize");
  return AFFON_ROCM_OK;
}

int affon_rocm_memcpy_h2d(affon_rocm_session* session, void* dst, const void* src, size_t bytes) {
  return copy(session, dst, src, bytes, hipMemcpyHostToDevice);
}

int affon_rocm_memcpy_d2h(affon_rocm_session* session, void* dst, const void* src, size_t bytes) {
  return copy(session, dst, src, bytes, hipMemcpyDeviceToHost);
}

int affon_rocm_memcpy_d2d(affon_rocm_session* session, void* dst, const void* src, size_t bytes) {
  return copy(session, dst, src, bytes, hipMemcpyDeviceToDevice);
}

int affon_rocm_synchronize(affon_rocm_session* session) {
  clear_error();
  int status = check_session(session);
  if (status != AFFON_ROCM_OK) return status;
  hipError_t e = hipStreamSynchronize(session->stream);
  if (e != hipSuccess) return hip_fail(e, "hipStreamSynchronize");
  return AFFON_ROCM_OK;
}

const char* affon_rocm_last_error(void) { return g_last_error.c_str(); }

int affon_rocm_quantized_matmul(affon_rocm_session* session, const affon_rocm_qmm_desc* desc) {
  clear_error();
  affon::QmmProblem p;
  int status = validate(desc, &p);
  if (status != AFFON_ROCM_OK) return status;
  const Candidate* c = nullptr;
  if ((status = select(desc, p, &c)) != AFFON_ROCM_OK) return status;
  if ((status = check_session(session)) != AFFON_ROCM_OK) return status;
  affon::Launch launch;
  launch.stream = session->stream;
  launch.workspace = session->workspace;
  hipError_t e = c->launch(p, launch);
  if (e != hipSuccess) return hip_fail(e, c->id);
  return AFFON_ROCM_OK;
}

int affon_rocm_quantized_matmul_noalloc(affon_rocm_session* session, const affon_rocm_qmm_desc* desc) {
  clear_error();
  affon::QmmProblem p;
  int status = validate(desc, &p);
  if (status != AFFON_ROCM_OK) return status;
  const Candidate* c = nullptr;
  if ((status = select(desc, p, &c)) != AFFON_ROCM_OK) return status;
  if ((status = check_session(session)) != AFFON_ROCM_OK) return status;
  void* fixed = nullptr;
  if (hipError_t e = scratch_on(session->device, &fixed); e != hipSuccess)
    return hip_fail(e, "hipGetSymbolAddress(scratch)");
  affon::Launch launch;
  launch.stream = session->stream;
  launch.fixed = fixed;
  launch.fixed_bytes = kNoAllocScratchBytes;
  hipError_t e = c->launch(p, launch);
  if (launch.fixed_short > 0)
    return fail(AFFON_ROCM_UNSUPPORTED,
                "%s needs %zu bytes of split-K scratch for this shape, more than the %zu bytes the no-allocation "
                "entry point holds; use affon_rocm_quantized_matmul",
                c->id, launch.fixed_short, kNoAllocScratchBytes);
  if (e != hipSuccess) return hip_fail(e, c->id);
  return AFFON_ROCM_OK;
}

int affon_rocm_read_floor(affon_rocm_session* session, const void* const* buffers, const uint64_t* bytes, int count,
                          void* sink) {
  clear_error();
  if (buffers == nullptr || bytes == nullptr || sink == nullptr || count < 1 || count > 4)
    return fail(AFFON_ROCM_INVALID_SHAPE, "read_floor needs 1 to 4 buffers, their sizes and a sink word");
  for (int i = 0; i < count; ++i) {
    if (buffers[i] == nullptr || reinterpret_cast<uintptr_t>(buffers[i]) % 16 != 0 || bytes[i] < 16)
      return fail(AFFON_ROCM_INVALID_SHAPE, "read_floor buffer %d is null, unaligned or shorter than 16 bytes", i);
  }
  int status = check_session(session);
  if (status != AFFON_ROCM_OK) return status;
  hipError_t e = affon::read_floor_launch(buffers, bytes, count, static_cast<uint32_t*>(sink), session->stream);
  if (e != hipSuccess) return hip_fail(e, "read_floor");
  return AFFON_ROCM_OK;
}

int affon_rocm_read_floor_geometry(affon_rocm_session* session, const void* buffer, uint64_t bytes, void* sink,
                                   uint64_t sink_bytes, const affon_rocm_floor_geometry* geometry) {
  clear_error();
  if (geometry == nullptr || buffer == nullptr || sink == nullptr)
    return fail(AFFON_ROCM_INVALID_SHAPE, "read_floor_geometry needs a buffer, a sink and a geometry");
  const affon_rocm_floor_geometry g = *geometry;
  if (reinterpret_cast<uintptr_t>(buffer) % 16 != 0 || reinterpret_cast<uintptr_t>(sink) % 8 != 0 || bytes < 16 ||
      bytes % 16 != 0)
    return fail(AFFON_ROCM_INVALID_SHAPE, "read_floor_geometry: buffer unaligned, or bytes not a positive multiple of 16");
  if (g.kib_per_wave != 1 && g.kib_per_wave != 2 && g.kib_per_wave != 4 && g.kib_per_wave != 8)
    return fail(AFFON_ROCM_INVALID_SHAPE, "read_floor_geometry: kib_per_wave must be 1, 2, 4 or 8");
  if (g.threads < 64 || g.threads > 1024 || g.threads % 64 != 0)
    return fail(AFFON_ROCM_INVALID_SHAPE, "read_floor_geometry: threads must be a multiple of 64 from 64 to 1024");
  if (g.valu_per_wave < 0 || g.valu_per_wave > 4096 || g.valu_per_wave % 8 != 0)
    return fail(AFFON_ROCM_INVALID_SHAPE, "read_floor_geometry: valu_per_wave must be a multiple of 8 from 0 to 4096");
  if (g.store_every < 0) return fail(AFFON_ROCM_INVALID_SHAPE, "read_floor_geometry: store_every must be >= 0");
  const uint64_t waves = affon::read_geometry_waves(bytes, g.kib_per_wave);
  const uint64_t need = g.store_every > 0 ? 8 * ((waves + g.store_every - 1) / g.store_every) : 4;
  if (sink_bytes < need)
    return fail(AFFON_ROCM_INVALID_SHAPE, "read_floor_geometry: sink holds %llu bytes, the stores need %llu",
                static_cast<unsigned long long>(sink_bytes), static_cast<unsigned long long>(need));
  int status = check_session(session);
  if (status != AFFON_ROCM_OK) return status;
  hipError_t e = affon::read_geometry_launch(buffer, bytes, static_cast<float*>(sink), g.kib_per_wave, g.threads,
                                             g.store_every, g.valu_per_wave, session->stream);
  if (e != hipSuccess) return hip_fail(e, "read_floor_geometry");
  return AFFON_ROCM_OK;
}

int affon_rocm_empty_launch(affon_rocm_session* session, uint32_t blocks, uint32_t threads) {
  clear_error();
  if (blocks < 1 || blocks > 0x7fffffffu || threads < 1 || threads > 1024)
    return fail(AFFON_ROCM_INVALID_SHAPE, "empty_launch: 1 to 2^31-1 workgroups of 1 to 1024 threads");
  int status = check_session(session);
  if (status != AFFON_ROCM_OK) return status;
  hipError_t e = affon::empty_launch(blocks, threads, session->stream);
  if (e != hipSuccess) return hip_fail(e, "empty_launch");
  return AFFON_ROCM_OK;
}

int affon_rocm_kernel_supports(const affon_rocm_qmm_desc* desc, const char* kernel, int* supported) {
  clear_error();
  if (kernel == nullptr || supported == nullptr)
    return fail(AFFON_ROCM_INVALID_SHAPE, "kernel_supports needs a kernel name and a result pointer");
  affon::QmmProblem p;
  int status = validate(desc, &p);
  if (status != AFFON_ROCM_OK) return status;
  static const struct {
    const char* name;
    bool (*guard)(const affon::QmmProblem&);
  } kGuards[] = {
      {"generic", affon::generic_supports}, {"gemv", affon::gemv_supports},     {"gemv1", affon::gemv1_supports},
      {"gemv_mfma", affon::gemv_mfma_supports}, {"mfma", affon::mfma_supports}, {"gemm_re", affon::re_gemm_supports},
      {"gemm_pair", affon::pair_supports},  {"gemm_re32", affon::re32_supports}, {"xgemm", affon::gemv_runs_xgemm},
  };
  for (const auto& g : kGuards) {
    if (std::strcmp(g.name, kernel) == 0) {
      *supported = g.guard(p) ? 1 : 0;
      return AFFON_ROCM_OK;
    }
  }
  return fail(AFFON_ROCM_INVALID_SHAPE, "kernel_supports: unknown kernel '%s'", kernel);
}

int affon_rocm_quantized_matmul_select(const affon_rocm_qmm_desc* desc, char* id, size_t cap) {
  clear_error();
  affon::QmmProblem p;
  int status = validate(desc, &p);
  if (status != AFFON_ROCM_OK) return status;
  const Candidate* c = nullptr;
  if ((status = select(desc, p, &c)) != AFFON_ROCM_OK) return status;
  if (id != nullptr && cap > 0) {
    std::strncpy(id, c->id, cap - 1);
    id[cap - 1] = '\0';
  }
  return AFFON_ROCM_OK;
}

}  // extern "C"

namespace {

// How a fused call runs: the first problem (the only one, or the gate
// projection), and for a two-launch SiLU gate the up projection, whose
// kernel multiplies silu(stored gate) into its output.
struct FusedPlan {
  affon::QmmProblem first, second;
  const Candidate* first_c = nullptr;
  const Candidate* second_c = nullptr;
  bool two = false;
};

bool same_layout(const affon_rocm_view& a, const affon_rocm_view& b) {
  return a.stride[0] == b.stride[0] && a.stride[1] == b.stride[1];
}

int plan_fused(const affon_rocm_qmm_desc* d, const affon_rocm_qmm_epilogue* e, FusedPlan* plan) {
  if (e == nullptr) return fail(AFFON_ROCM_INVALID_SHAPE, "quantized_matmul epilogue is null");
  int status = validate(d, &plan->first);
  if (status != AFFON_ROCM_OK) return status;
  affon::QmmProblem& p = plan->first;
  switch (e->kind) {
    case AFFON_ROCM_EPILOGUE_NONE:
      return select(d, p, &plan->first_c);
    case AFFON_ROCM_EPILOGUE_BIAS: {
      const int esize = element_size(e->bias_dtype);
      if (e->bias == nullptr || !is_float_dtype(e->bias_dtype))
        return fail(AFFON_ROCM_INVALID_SHAPE, "quantized_matmul output bias must be an f32/bf16 vector");
      if (e->bias_bytes / static_cast<size_t>(esize) < static_cast<size_t>(p.N) ||
          reinterpret_cast<uintptr_t>(e->bias) % static_cast<uintptr_t>(esize) != 0)
        return fail(AFFON_ROCM_INVALID_SHAPE, "quantized_matmul output bias needs N aligned elements");
      p.epi.kind = affon::kEpiBias;
      p.epi.bias = static_cast<const uint8_t*>(e->bias);
      p.epi.bias_bf16 = e->bias_dtype == AFFON_ROCM_BF16;
      return select(d, p, &plan->first_c);
    }
    case AFFON_ROCM_EPILOGUE_SILU_GATE: {
      const affon_rocm_view* gate[3] = {&d->packed, &d->scales, &d->biases};
      const affon_rocm_view* up[3] = {&e->up_packed, &e->up_scales, &e->up_biases};
      const char* names[3] = {"up packed", "up scales", "up biases"};
      for (int i = 0; i < 3; ++i) {
        if (up[i]->dtype != gate[i]->dtype || up[i]->shape[0] != gate[i]->shape[0] ||
            up[i]->shape[1] != gate[i]->shape[1])
          return fail(AFFON_ROCM_INVALID_SHAPE, "quantized_matmul %s must match the gate projection's shape and dtype",
                      names[i]);
        if ((status = check_view(*up[i], names[i])) != AFFON_ROCM_OK) return status;
      }
      affon::QmmProblem& q = plan->second;
      q = p;
      q.w = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(e->up_packed.data) +
                                              e->up_packed.byte_offset);
      q.ws0 = e->up_packed.stride[0];
      q.ws1 = e->up_packed.stride[1];
      q.s = static_cast<const uint8_t*>(e->up_scales.data) + e->up_scales.byte_offset;
      q.ss0 = e->up_scales.stride[0];
      q.ss1 = e->up_scales.stride[1];
      q.b = static_cast<const uint8_t*>(e->up_biases.data) + e->up_biases.byte_offset;
      q.bs0 = e->up_biases.stride[0];
      q.bs1 = e->up_biases.stride[1];
      if ((status = select(d, p, &plan->first_c)) != AFFON_ROCM_OK) return status;
      // One launch when the gate's kernel pairs rows of both projections.
      affon::QmmProblem paired = p;
      paired.epi.kind = affon::kEpiSiluPair;
      paired.epi.w2 = q.w;
      paired.epi.s2 = q.s;
      paired.epi.b2 = q.b;
      if (plan->first_c->impl == AFFON_ROCM_IMPL_GEMV && same_layout(d->packed, e->up_packed) &&
          same_layout(d->scales, e->up_scales) && same_layout(d->biases, e->up_biases) &&
          affon::gemv_pair_supports(paired)) {
        p = paired;
        return AFFON_ROCM_OK;
      }
      plan->two = true;
      q.epi.kind = affon::kEpiGateMul;
      return select(d, q, &plan->second_c);
    }
    default:
      return fail(AFFON_ROCM_INVALID_SHAPE, "quantized_matmul unknown epilogue %d", e->kind);
  }
}

std::string fused_text(const FusedPlan& plan);
int copy_id(const std::string& text, char* id, size_t cap);

}  // namespace

extern "C" {

int affon_rocm_quantized_matmul_fused(affon_rocm_session* session, const affon_rocm_qmm_desc* desc,
                                      const affon_rocm_qmm_epilogue* epilogue) {
  clear_error();
  FusedPlan plan;
  int status = plan_fused(desc, epilogue, &plan);
  if (status != AFFON_ROCM_OK) return status;
  if ((status = check_session(session)) != AFFON_ROCM_OK) return status;
  affon::Launch launch;
  launch.stream = session->stream;
  launch.workspace = session->workspace;
  hipError_t e = plan.first_c->launch(plan.first, launch);
  if (e != hipSuccess) return hip_fail(e, plan.first_c->id);
  if (plan.two) {
    e = plan.second_c->launch(plan.second, launch);
    if (e != hipSuccess) return hip_fail(e, plan.second_c->id);
  }
  return AFFON_ROCM_OK;
}

int affon_rocm_quantized_matmul_fused_select(const affon_rocm_qmm_desc* desc, const affon_rocm_qmm_epilogue* epilogue,
                                             char* id, size_t cap) {
  clear_error();
  FusedPlan plan;
  int status = plan_fused(desc, epilogue, &plan);
  if (status != AFFON_ROCM_OK) return status;
  return copy_id(fused_text(plan), id, cap);
}

}  // extern "C"

namespace {

bool same_view(const affon_rocm_view& a, const affon_rocm_view& b) {
  return a.data == b.data && a.byte_offset == b.byte_offset && a.shape[0] == b.shape[0] && a.shape[1] == b.shape[1] &&
         a.stride[0] == b.stride[0] && a.stride[1] == b.stride[1] && a.dtype == b.dtype;
}

// A grouped call: every member's plan, and whether they run as one launch.
struct GroupPlan {
  FusedPlan members[affon::kMaxGroup];
  std::vector<FusedPlan> many;  // more members than one launch takes
  size_t count = 0;
  bool one_launch = false;
  int one_impl = 0;  // the candidate whose kernel runs the whole group
  const FusedPlan& at(size_t i) const { return count <= affon::kMaxGroup ? members[i] : many[i]; }
};

int plan_grouped(const affon_rocm_qmm_desc* descs, const affon_rocm_qmm_epilogue* epilogues, size_t count,
                 GroupPlan* plan) {
  if (descs == nullptr || count == 0)
    return fail(AFFON_ROCM_INVALID_SHAPE, "grouped quantized_matmul needs at least one descriptor");
  if (count > affon::kMaxGroup) plan->many.resize(count);
  plan->count = count;
  affon_rocm_qmm_epilogue none;
  std::memset(&none, 0, sizeof(none));
  none.kind = AFFON_ROCM_EPILOGUE_NONE;
  for (size_t i = 0; i < count; ++i) {
    const affon_rocm_qmm_desc& d = descs[i];
    if (i > 0 && (!same_view(d.input, descs[0].input) || d.bits != descs[0].bits ||
                  d.group_size != descs[0].group_size || d.implementation != descs[0].implementation ||
                  d.numerical_policy != descs[0].numerical_policy))
      return fail(AFFON_ROCM_INVALID_SHAPE, "grouped quantized_matmul descriptors must share the input and options");
    const affon_rocm_qmm_epilogue* e = epilogues != nullptr ? &epilogues[i] : &none;
    if (e->kind != AFFON_ROCM_EPILOGUE_NONE && e->kind != AFFON_ROCM_EPILOGUE_BIAS)
      return fail(AFFON_ROCM_INVALID_SHAPE, "grouped quantized_matmul takes no epilogue or an output bias per call");
    FusedPlan& member = count <= affon::kMaxGroup ? plan->members[i] : plan->many[i];
    int status = plan_fused(&d, e, &member);
    if (status != AFFON_ROCM_OK) return status;
  }
  if (count >= 2 && count <= affon::kMaxGroup) {
    affon::QmmProblem problems[affon::kMaxGroup];
    const int impl = plan->members[0].first_c->impl;
    bool same = true;
    for (size_t i = 0; i < count; ++i) {
      problems[i] = plan->members[i].first;
      same = same && plan->members[i].first_c->impl == impl;
    }
    const int n = static_cast<int>(count);
    if (same && impl == AFFON_ROCM_IMPL_GEMV)
      plan->one_launch = affon::gemv_group_supports(problems, n);
    else if (same && impl == AFFON_ROCM_IMPL_GEMV_MFMA)
      plan->one_launch = affon::gemv_mfma_group_supports(problems, n);
    plan->one_impl = impl;
  }
  return AFFON_ROCM_OK;
}

std::string fused_text(const FusedPlan& plan) {
  std::string text = plan.first_c->id;
  switch (plan.first.epi.kind) {
    case affon::kEpiBias: text += "[bias]"; break;
    case affon::kEpiSiluPair: text += "[silu_gate]"; break;
    default: break;
  }
  if (plan.two) text += std::string(";") + plan.second_c->id + "[gate_mul]";
  return text;
}

int copy_id(const std::string& text, char* id, size_t cap) {
  if (id != nullptr && cap > 0) {
    std::strncpy(id, text.c_str(), cap - 1);
    id[cap - 1] = '\0';
  }
  return AFFON_ROCM_OK;
}

}  // namespace

extern "C" {

int affon_rocm_quantized_matmul_grouped(affon_rocm_session* session, const affon_rocm_qmm_desc* descs,
                                        const affon_rocm_qmm_epilogue* epilogues, size_t count) {
  clear_error();
  GroupPlan plan;
  int status = plan_grouped(descs, epilogues, count, &plan);
  if (status != AFFON_ROCM_OK) return status;
  if ((status = check_session(session)) != AFFON_ROCM_OK) return status;
  affon::Launch launch;
  launch.stream = session->stream;
  launch.workspace = session->workspace;
  if (plan.one_launch) {
    affon::QmmProblem problems[affon::kMaxGroup];
    for (size_t i = 0; i < count; ++i) problems[i] = plan.members[i].first;
    const int n = static_cast<int>(count);
    hipError_t e = plan.one_impl == AFFON_ROCM_IMPL_GEMV ? affon::gemv_group_launch(problems, n, launch)
                                                         : affon::gemv_mfma_group_launch(problems, n, launch);
    if (e != hipSuccess) return hip_fail(e, "grouped quantized_matmul");
    return AFFON_ROCM_OK;
  }
  for (size_t i = 0; i < count; ++i) {
    const FusedPlan& member = plan.at(i);
    hipError_t e = member.first_c->launch(member.first, launch);
    if (e != hipSuccess) return hip_fail(e, member.first_c->id);
  }
  return AFFON_ROCM_OK;
}

int affon_rocm_quantized_matmul_grouped_select(const affon_rocm_qmm_desc* descs,
                                               const affon_rocm_qmm_epilogue* epilogues, size_t count, char* id,
                                               size_t cap) {
  clear_error();
  GroupPlan plan;
  int status = plan_grouped(descs, epilogues, count, &plan);
  if (status != AFFON_ROCM_OK) return status;
  if (plan.one_launch) {
    bool bias = false;
    for (size_t i = 0; i < count; ++i) bias = bias || plan.members[i].first.epi.kind == affon::kEpiBias;
    return copy_id(std::string(plan.members[0].first_c->id) + "[grouped:" + std::to_string(count) +
                       (bias ? ",bias]" : "]"),
                   id, cap);
  }
  std::string text;
  for (size_t i = 0; i < count; ++i) text += (i ? ";" : "") + fused_text(plan.at(i));
  return copy_id(text, id, cap);
}

const char* affon_rocm_quantized_matmul_capabilities(void) {
  static const char* kJson =
      "["
      "{\"id\":\"rocm_quantized_matmul.mfma\",\"version\":1,\"numerical_class\":\"approximate\","
      "\"guard\":\"gfx950; bf16 input; group_size % 32 == 0; K % 64 == 0; unit inner strides; M >= 64 when auto\","
      "\"note\":\"decoded weights rounded to bf16 in LDS, bf16 MFMA, f32 accumulation\"},"
      "{\"id\":\"rocm_quantized_matmul.gemv_mfma\",\"version\":1,\"numerical_class\":\"reassociated\","
      "\"guard\":\"gfx950; bf16 input; group_size a power of two >= 64; K % 256 == 0; unit inner strides; M >= 2 when auto (rows beyond 32 in row tiles)\","
      "\"note\":\"integer codes exact in bf16, per-group scale and bias applied in f32\"},"
      "{\"id\":\"rocm_quantized_matmul.gemv\",\"version\":1,\"numerical_class\":\"reassociated\","
      "\"guard\":\"gfx950; group_size % (32/bits) == 0; unit inner strides; aligned rows\","
      "\"note\":\"one row and few passes: VALU decode; other batches with groups of 32s: matrix cores, codes exact in "
      "bf16, f32 activations in three bf16 planes; f32 accumulation, per-group scale and bias applied in f32\"},"
      "{\"id\":\"rocm_quantized_matmul.generic\",\"version\":1,\"numerical_class\":\"exact\","
      "\"guard\":\"gfx950; any strides, byte offsets and group sizes\","
      "\"note\":\"ordered f32 loop per output, separately rounded products and sums\"}"
      "]";
  return kJson;
}

int affon_rocm_quantize(affon_rocm_session* session, const void* weights, int32_t weight_dtype, int64_t rows,
                        int64_t columns, uint32_t bits, uint32_t group_size, uint32_t* packed, void* scales,
                        void* biases, int32_t param_dtype) {
  clear_error();
  if (bits != 2 && bits != 4 && bits != 8) return fail(AFFON_ROCM_INVALID_SHAPE, "quantize bits must be 2, 4, or 8");
  if (group_size == 0) return fail(AFFON_ROCM_INVALID_SHAPE, "quantize group_size must be a positive integer");
  if (!is_float_dtype(weight_dtype) || !is_float_dtype(param_dtype))
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantize requires f32/bf16 weights and f32/bf16 parameters");
  const int64_t per_word = 32 / static_cast<int64_t>(bits);
  if (rows <= 0 || columns <= 0 || columns % per_word != 0 || columns % static_cast<int64_t>(group_size) != 0)
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantize columns must divide into complete words and groups");
  uint64_t count = 0;
  if (!mul_ok(static_cast<uint64_t>(rows), static_cast<uint64_t>(columns), &count) || count > (uint64_t(1) << 60))
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantize size overflows");
  if (weights == nullptr || packed == nullptr || scales == nullptr || biases == nullptr)
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantize buffer is null");
  int status = check_session(session);
  if (status != AFFON_ROCM_OK) return status;
  hipError_t e = affon::quantize_launch(weights, weight_dtype, rows, columns, static_cast<int>(bits), group_size,
                                        packed, scales, biases, param_dtype, session->stream);
  if (e != hipSuccess) return hip_fail(e, "quantize");
  return AFFON_ROCM_OK;
}

int affon_rocm_dequantize(affon_rocm_session* session, const uint32_t* packed, const void* scales, const void* biases,
                          int32_t param_dtype, int64_t rows, int64_t columns, uint32_t bits, uint32_t group_size,
                          void* out, int32_t out_dtype) {
  clear_error();
  if (bits != 2 && bits != 4 && bits != 8)
    return fail(AFFON_ROCM_INVALID_SHAPE, "dequantize bits must be 2, 4, or 8");
  if (group_size == 0) return fail(AFFON_ROCM_INVALID_SHAPE, "dequantize group_size must be a positive integer");
  if (!is_float_dtype(param_dtype) || !is_float_dtype(out_dtype))
    return fail(AFFON_ROCM_INVALID_SHAPE, "dequantize requires f32/bf16 parameters and output");
  const int64_t per_word = 32 / static_cast<int64_t>(bits);
  if (rows <= 0 || columns <= 0 || columns % per_word != 0 || columns % static_cast<int64_t>(group_size) != 0)
    return fail(AFFON_ROCM_INVALID_SHAPE, "dequantize columns must divide into complete words and groups");
  uint64_t count = 0;
  if (!mul_ok(static_cast<uint64_t>(rows), static_cast<uint64_t>(columns), &count) || count > (uint64_t(1) << 60))
    return fail(AFFON_ROCM_INVALID_SHAPE, "dequantize size overflows");
  if (packed == nullptr || scales == nullptr || biases == nullptr || out == nullptr)
    return fail(AFFON_ROCM_INVALID_SHAPE, "dequantize buffer is null");
  int status = check_session(session);
  if (status != AFFON_ROCM_OK) return status;
  hipError_t e = affon::dequantize_launch(packed, scales, biases, param_dtype, rows, columns, static_cast<int>(bits),
                                          group_size, out, out_dtype, session->stream);
  if (e != hipSuccess) return hip_fail(e, "dequantize");
  return AFFON_ROCM_OK;
}

static int check_rows(const void* x, int32_t dtype, int64_t rows, int64_t cols, const void* out, const char* op) {
  if (!is_float_dtype(dtype)) return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires an f32 or bf16 tensor", op);
  if (rows <= 0 || cols <= 0) return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires a non-empty rank-two tensor", op);
  uint64_t count = 0;
  // Workgroups of rows stride over what a grid does not hold; one thread per
  // element (index_select of columns) must stay within 2^31 workgroups.
  if (!mul_ok(static_cast<uint64_t>(rows), static_cast<uint64_t>(cols), &count) || count > (uint64_t(1) << 40) ||
      rows > (int64_t(1) << 32))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s size overflows", op);
  if (x == nullptr || out == nullptr) return fail(AFFON_ROCM_INVALID_SHAPE, "%s buffer is null", op);
  return AFFON_ROCM_OK;
}

int affon_rocm_rms_norm(affon_rocm_session* session, const void* x, int32_t dtype, int64_t rows, int64_t cols,
                        float epsilon, void* out) {
  clear_error();
  int status = check_rows(x, dtype, rows, cols, out, "rms_norm");
  if (status != AFFON_ROCM_OK) return status;
  // program.ts:578-579: a finite, positive epsilon.
  if (!(epsilon > 0.0f) || epsilon == std::numeric_limits<float>::infinity())
    return fail(AFFON_ROCM_INVALID_SHAPE, "invalid rms_norm options: epsilon must be finite and positive");
  if ((status = check_session(session)) != AFFON_ROCM_OK) return status;
  hipError_t e = affon::rms_norm_launch(x, dtype, rows, cols, epsilon, out, session->stream);
  if (e != hipSuccess) return hip_fail(e, "rms_norm");
  return AFFON_ROCM_OK;
}

int affon_rocm_softmax(affon_rocm_session* session, const void* x, int32_t dtype, int64_t rows, int64_t cols,
                       void* out) {
  clear_error();
  int status = check_rows(x, dtype, rows, cols, out, "softmax");
  if (status != AFFON_ROCM_OK) return status;
  if ((status = check_session(session)) != AFFON_ROCM_OK) return status;
  affon::Launch launch;
  launch.stream = session->stream;
  launch.workspace = session->workspace;
  hipError_t e = affon::softmax_launch(x, dtype, rows, cols, out, launch);
  if (e != hipSuccess) return hip_fail(e, "softmax");
  return AFFON_ROCM_OK;
}

int affon_rocm_index_select(affon_rocm_session* session, const void* x, int32_t dtype, int64_t rows, int64_t cols,
                            int32_t axis, const int64_t* index, int64_t count, void* out) {
  clear_error();
  int status = check_rows(x, dtype, rows, cols, out, "index_select");
  if (status != AFFON_ROCM_OK) return status;
  if (axis != 0 && axis != 1) return fail(AFFON_ROCM_INVALID_SHAPE, "index_select axis must be 0 or 1");
  if (count <= 0 || index == nullptr) return fail(AFFON_ROCM_INVALID_SHAPE, "index_select requires indices");
  uint64_t total = 0;
  if (!mul_ok(static_cast<uint64_t>(count), static_cast<uint64_t>(axis == 0 ? cols : rows), &total) ||
      total > (uint64_t(1) << 38))
    return fail(AFFON_ROCM_INVALID_SHAPE, "index_select size overflows");
  if ((status = check_session(session)) != AFFON_ROCM_OK) return status;
  hipError_t e = affon::index_select_launch(x, dtype, rows, cols, axis, index, count, out, session->stream);
  if (e != hipSuccess) return hip_fail(e, "index_select");
  return AFFON_ROCM_OK;
}

// ---- drafted tokens over a paged cache, and the norms between blocks ----

namespace {

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// A view of a rank-two operand [rows, cols] with unit inner stride.
int check_matrix(const affon_rocm_view& v, int64_t rows, int64_t cols, const char* name, const char* op) {
  if (v.shape[0] != rows || v.shape[1] != cols)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s %s must be [%lld, %lld]", op, name, static_cast<long long>(rows),
                static_cast<long long>(cols));
  if (cols > 1 && v.stride[1] != 1)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s %s must have a unit inner stride", op, name);
  if (!aligned(v.data, element_size(v.dtype)))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s %s is not element aligned", op, name);
  return check_view(v, name, op);
}

const uint8_t* origin(const affon_rocm_view& v) { return static_cast<const uint8_t*>(v.data) + v.byte_offset; }

constexpr int64_t kMaxInt = std::numeric_limits<int32_t>::max();

// The product of positive factors, or false where one is not positive or it passes 2^40.
bool extent(std::initializer_list<int64_t> factors, uint64_t* out) {
  *out = 1;
  for (int64_t f : factors)
    if (f <= 0 || !mul_ok(*out, static_cast<uint64_t>(f), out) || *out > (uint64_t(1) << 40)) return false;
  return true;
}

// `layer`: the one that is used, or -1 for all.
int check_cache(const affon_rocm_kv_cache* c, int64_t layer, const char* op, affon::PagedCache* out) {
  if (c == nullptr) return fail(AFFON_ROCM_INVALID_SHAPE, "%s cache is null", op);
  if (!is_float_dtype(c->dtype)) return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires an f32 or bf16 cache", op);
  uint64_t count = 0;
  if (!extent({c->layers, c->pages, c->kv_heads, c->page_size, c->head_dim}, &count))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s cache has an empty dimension or its size overflows", op);
  if (c->page_size % 16 != 0 || c->page_size > 65536)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s page_size must be a multiple of 16, at most 65536", op);
  if (c->head_dim % 8 != 0 || c->head_dim > 256)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s head_dim must be a multiple of 8, at most 256", op);
  if (c->layers > kMaxInt || c->pages > kMaxInt || c->kv_heads > 65535)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s cache size overflows", op);
  const uint64_t bytes = count * static_cast<uint64_t>(element_size(c->dtype));
  if (c->keys == nullptr || c->values == nullptr || c->bytes < bytes)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s cache memory is smaller than its shape", op);
  if (!aligned(c->keys, 16) || !aligned(c->values, 16))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s cache must be 16-byte aligned", op);
  if (layer < -1 || layer >= c->layers) return fail(AFFON_ROCM_INVALID_SHAPE, "%s layer is out of range", op);
  out->layer_bytes = static_cast<int64_t>(bytes / static_cast<uint64_t>(c->layers));
  const int64_t at = layer > 0 ? layer * out->layer_bytes : 0;
  out->keys = static_cast<uint8_t*>(c->keys) + at;
  out->values = static_cast<uint8_t*>(c->values) + at;
  out->dtype = c->dtype;
  out->layers = layer < 0 ? static_cast<int>(c->layers) : 1;
  out->pages = static_cast<int>(c->pages);
  out->kv_heads = static_cast<int>(c->kv_heads);
  out->page_size = static_cast<int>(c->page_size);
  out->head_dim = static_cast<int>(c->head_dim);
  return AFFON_ROCM_OK;
}

int check_batch(const affon_rocm_draft_batch* b, const affon::PagedCache& cache, const char* op,
                affon::DraftBatch* out) {
  if (b == nullptr) return fail(AFFON_ROCM_INVALID_SHAPE, "%s batch is null", op);
  const affon_rocm_view& t = b->page_table;
  if (t.dtype != AFFON_ROCM_U32) return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires a u32 page table", op);
  int status = check_matrix(t, t.shape[0], t.shape[1], "page table", op);
  if (status != AFFON_ROCM_OK) return status;
  uint64_t rows = 0, tokens = 0;
  if (!extent({t.shape[0], b->rows}, &rows) || rows > static_cast<uint64_t>(kMaxInt / 2))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires at least one row per sequence, and their number to fit 30 bits", op);
  if (!extent({t.shape[1], cache.page_size}, &tokens) || tokens + static_cast<uint64_t>(b->rows) > static_cast<uint64_t>(kMaxInt))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s page table covers too many tokens", op);
  if (b->lengths == nullptr || !aligned(b->lengths, 4) || !aligned(b->counts, 4))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires u32 lengths", op);
  out->sequences = static_cast<int>(t.shape[0]);
  out->rows = static_cast<int>(b->rows);
  out->table = reinterpret_cast<const uint32_t*>(origin(t));
  out->table_stride = t.stride[0];
  out->capacity = static_cast<uint32_t>(tokens);
  out->lengths = b->lengths;
  out->counts = b->counts;
  return AFFON_ROCM_OK;
}

// The queries of a batch: [B*T, heads*head_dim], heads a multiple of kv_heads; and (`has_output`) an output of their shape.
int check_query(const affon_rocm_view& q, const affon::PagedCache& cache, const affon::DraftBatch& batch,
                const void* output, size_t output_bytes, const char* op, int* heads, bool has_output = true) {
  const int64_t rows = static_cast<int64_t>(batch.sequences) * batch.rows;
  const int64_t unit = static_cast<int64_t>(cache.kv_heads) * cache.head_dim;
  if (q.shape[1] <= 0 || q.shape[1] % unit != 0 || q.shape[1] / cache.head_dim > 65535)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s query width must be a multiple of kv_heads * head_dim", op);
  const int status = check_matrix(q, rows, q.shape[1], "query", op);
  if (status != AFFON_ROCM_OK) return status;
  uint64_t count = 0;
  if (!extent({rows, q.shape[1]}, &count)) return fail(AFFON_ROCM_INVALID_SHAPE, "%s query size overflows", op);
  *heads = static_cast<int>(q.shape[1] / cache.head_dim);
  if (!has_output) return AFFON_ROCM_OK;
  if (output == nullptr || output_bytes < count * static_cast<uint64_t>(element_size(cache.dtype)) ||
      !aligned(output, element_size(cache.dtype)))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s output buffer is smaller than the query", op);
  return AFFON_ROCM_OK;
}

affon::Rows rows_of_view(const affon_rocm_view& v) {
  if (v.data == nullptr) return affon::Rows{nullptr, 0, 0, 0};
  const int64_t size = element_size(v.dtype);
  return affon::rows_of(origin(v), v.shape[0], v.shape[1] * size, v.stride[0] * size);
}

affon::Rows words(const void* data, int64_t count) { return affon::rows_of(data, 1, count * 4, 0); }

// Whether `out` shares memory with the cache, the batch or one of `others`.
bool meets(const affon::Rows& out, const affon_rocm_kv_cache& cache, const affon_rocm_draft_batch& batch,
           const affon::DraftBatch& b, std::initializer_list<affon::Rows> others) {
  const int64_t cache_bytes = cache.layers * cache.pages * cache.kv_heads * cache.page_size * cache.head_dim *
                              element_size(cache.dtype);
  for (const auto& held : {affon::rows_of(cache.keys, 1, cache_bytes, 0), affon::rows_of(cache.values, 1, cache_bytes, 0),
                           rows_of_view(batch.page_table), words(b.lengths, b.sequences), words(b.counts, b.sequences)})
    if (affon::rows_meet(held, out)) return true;
  for (const auto& other : others)
    if (affon::rows_meet(other, out)) return true;
  return false;
}

// The output of the queries' shape: it may be the query itself, as whoever
// writes a value there has read it before, and otherwise overlaps nothing.
int check_output(const void* output, const affon_rocm_view& query, const affon_rocm_kv_cache& cache,
                 const affon_rocm_draft_batch& batch, const affon::DraftBatch& b, const char* op,
                 std::initializer_list<affon::Rows> others) {
  const int64_t bytes = query.shape[1] * element_size(cache.dtype);
  const affon::Rows out = affon::rows_of(output, query.shape[0], bytes, bytes);
  const affon::Rows q = rows_of_view(query);
  const bool clear = (!affon::rows_meet(q, out) || affon::same_rows(q, out)) && !meets(out, cache, batch, b, others);
  if (!clear) return fail(AFFON_ROCM_INVALID_SHAPE, "%s output overlaps an operand that it is not", op);
  return AFFON_ROCM_OK;
}

// An append's operands, but for what its output overlaps.
int check_append(const affon_rocm_kv_cache* cache, const affon_rocm_draft_batch* batch, const affon_rocm_append_desc* d,
                 const char* op, affon::AppendProblem* out) {
  affon::AppendProblem& p = *out;
  if (d->layer < 0) return fail(AFFON_ROCM_INVALID_SHAPE, "%s layer is out of range", op);
  int status = check_cache(cache, d->layer, op, &p.cache);
  if (status != AFFON_ROCM_OK || (status = check_batch(batch, p.cache, op, &p.batch)) != AFFON_ROCM_OK) return status;
  if (!is_float_dtype(d->query.dtype) || d->key.dtype != d->query.dtype || d->value.dtype != d->query.dtype)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires query, key and value of one type, f32 or bf16", op);
  if ((status = check_query(d->query, p.cache, p.batch, d->output, d->output_bytes, op, &p.heads)) != AFFON_ROCM_OK)
    return status;
  const int64_t rows = d->query.shape[0], width = static_cast<int64_t>(p.cache.kv_heads) * p.cache.head_dim;
  if ((status = check_matrix(d->key, rows, width, "key", op)) != AFFON_ROCM_OK ||
      (status = check_matrix(d->value, rows, width, "value", op)) != AFFON_ROCM_OK)
    return status;
  if (d->rotary_dim < 2 || d->rotary_dim % 2 != 0 || d->rotary_dim > p.cache.head_dim)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s rotary_dim must be even, and at most head_dim", op);
  if (d->rotary == nullptr || !aligned(d->rotary, 4) || !aligned(d->positions, 4) || d->rotary_rows <= 0 ||
      d->rotary_rows > kMaxInt)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires an f32 rotary table", op);
  p.query = origin(d->query);
  p.key = origin(d->key);
  p.value = origin(d->value);
  p.query_stride = d->query.stride[0];
  p.key_stride = d->key.stride[0];
  p.value_stride = d->value.stride[0];
  p.x_dtype = d->query.dtype;
  p.positions = d->positions;
  p.rotary = d->rotary;
  p.rotary_rows = static_cast<uint32_t>(d->rotary_rows);
  p.rotary_dim = static_cast<int>(d->rotary_dim);
  p.interleaved = d->interleaved != 0;
  p.out = static_cast<uint8_t*>(d->output);
  return AFFON_ROCM_OK;
}

// An attention's operands but for its output: query, mask, scale and layer.
int check_attention(const affon_rocm_kv_cache* cache, const affon_rocm_draft_batch* batch, const affon_rocm_view& query,
                    const affon_rocm_view& mask, float scale, int64_t layer, const void* output, size_t output_bytes,
                    const char* op, affon::AttentionProblem* out, bool has_output = true) {
  affon::AttentionProblem& p = *out;
  if (layer < 0) return fail(AFFON_ROCM_INVALID_SHAPE, "%s layer is out of range", op);
  int status = check_cache(cache, layer, op, &p.cache);
  if (status != AFFON_ROCM_OK || (status = check_batch(batch, p.cache, op, &p.batch)) != AFFON_ROCM_OK) return status;
  if (query.dtype != p.cache.dtype)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires query and cache of one type", op);
  if ((status = check_query(query, p.cache, p.batch, output, output_bytes, op, &p.heads, has_output)) != AFFON_ROCM_OK)
    return status;
  if (mask.data != nullptr) {
    if (mask.dtype != AFFON_ROCM_U32 || mask.shape[1] < (p.batch.rows + 31) / 32)
      return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires a u32 mask with a bit for every row of a sequence", op);
    if ((status = check_matrix(mask, query.shape[0], mask.shape[1], "mask", op)) != AFFON_ROCM_OK) return status;
    p.mask = reinterpret_cast<const uint32_t*>(origin(mask));
    p.mask_stride = mask.stride[0];
  }
  if (!(scale - scale == 0.0f)) return fail(AFFON_ROCM_INVALID_SHAPE, "%s scale must be finite", op);
  p.query = origin(query);
  p.query_stride = query.stride[0];
  p.scale = scale;
  return AFFON_ROCM_OK;
}

// Gathered weights f32 [layers, B, kv_heads, columns * page_size].
int check_weights(const affon_rocm_kv_cache& cache, const affon::DraftBatch& b, const void* weights, size_t bytes,
                  const char* op, affon::Rows* out) {
  uint64_t count = 0;
  if (!extent({cache.layers, b.sequences, cache.kv_heads, static_cast<int64_t>(b.capacity)}, &count))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s weights' size overflows", op);
  if (weights == nullptr || !aligned(weights, 4) || bytes < count * 4)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires f32 weights [layers, sequences, kv_heads, columns * page_size]", op);
  *out = affon::rows_of(weights, 1, static_cast<int64_t>(count) * 4, 0);
  return AFFON_ROCM_OK;
}

// A commit's operands: the cache's every layer, and the accepted tokens' path.
int check_commit(const affon_rocm_kv_cache* cache, const affon_rocm_draft_batch* batch, const affon_rocm_view* path,
                 const uint32_t* accepted, const char* op, affon::PagedCache* c, affon::DraftBatch* b) {
  int status = check_cache(cache, -1, op, c);
  if (status != AFFON_ROCM_OK || (status = check_batch(batch, *c, op, b)) != AFFON_ROCM_OK) return status;
  if (path == nullptr || path->dtype != AFFON_ROCM_U32 || path->shape[1] > b->rows)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires a u32 path of at most the batch's rows", op);
  if ((status = check_matrix(*path, b->sequences, path->shape[1], "path", op)) != AFFON_ROCM_OK) return status;
  if (accepted == nullptr || !aligned(accepted, 4))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires u32 counts of accepted tokens", op);
  return AFFON_ROCM_OK;
}

}  // namespace

int affon_rocm_cache_append(affon_rocm_session* session, const affon_rocm_kv_cache* cache,
                            const affon_rocm_draft_batch* batch, const affon_rocm_append_desc* d) {
  clear_error();
  const char* op = "cache_append";
  if (d == nullptr) return fail(AFFON_ROCM_INVALID_SHAPE, "%s descriptor is null", op);
  affon::AppendProblem p{};
  int status = check_append(cache, batch, d, op, &p);
  if (status != AFFON_ROCM_OK) return status;
  const int64_t rows = d->query.shape[0];
  if ((status = check_session(session)) != AFFON_ROCM_OK ||
      (status = check_output(d->output, d->query, *cache, *batch, p.batch, op,
                             {rows_of_view(d->key), rows_of_view(d->value), words(d->positions, rows),
                              words(d->rotary, d->rotary_rows * d->rotary_dim)})) != AFFON_ROCM_OK)
    return status;
  const hipError_t e = affon::append_launch(p, session->stream);
  if (e != hipSuccess) return hip_fail(e, op);
  return AFFON_ROCM_OK;
}

int affon_rocm_cache_append_normed(affon_rocm_session* session, const affon_rocm_kv_cache* cache,
                                   const affon_rocm_draft_batch* batch, const affon_rocm_append_desc* d,
                                   const affon_rocm_head_norm* norm) {
  clear_error();
  const char* op = "cache_append";
  if (d == nullptr || norm == nullptr) return fail(AFFON_ROCM_INVALID_SHAPE, "%s descriptor is null", op);
  affon::AppendNormProblem q{};
  int status = check_append(cache, batch, d, op, &q.base);
  if (status != AFFON_ROCM_OK) return status;
  const affon::AppendProblem& p = q.base;
  const int64_t rows = d->query.shape[0], D = p.cache.head_dim;
  affon::Rows weights[2];
  for (int k = 0; k < 2; ++k) {
    affon::HeadNorm& n = k == 0 ? q.query_norm : q.key_norm;
    n.weight = static_cast<const uint8_t*>(k == 0 ? norm->query_weight : norm->key_weight);
    n.stride = k == 0 ? norm->query_weight_stride : norm->key_weight_stride;
    n.dtype = k == 0 ? norm->query_weight_dtype : norm->key_weight_dtype;
    weights[k] = words(nullptr, 0);
    if (n.weight == nullptr) continue;
    if (!is_float_dtype(n.dtype) || (n.stride != 0 && n.stride != D) || !aligned(n.weight, element_size(n.dtype)))
      return fail(AFFON_ROCM_INVALID_SHAPE, "%s norm weights must be f32 or bf16, of one head or of each", op);
    const int64_t heads = n.stride == 0 ? 1 : k == 0 ? p.heads : p.cache.kv_heads;
    weights[k] = affon::rows_of(n.weight, 1, heads * D * element_size(n.dtype), 0);
  }
  q.epsilon = norm->epsilon;
  if (!(q.epsilon > 0.0f) || q.epsilon == std::numeric_limits<float>::infinity())
    return fail(AFFON_ROCM_INVALID_SHAPE, "invalid cache_append options: epsilon must be finite and positive");
  q.axes = norm->axes;
  if (q.axes < 1 || q.axes > 4) return fail(AFFON_ROCM_INVALID_SHAPE, "%s takes positions of one to four axes", op);
  for (int j = 0; j < p.rotary_dim / 2; ++j) {
    if (norm->axis[j] >= q.axes) return fail(AFFON_ROCM_INVALID_SHAPE, "%s pair has an axis that the positions have not", op);
    q.axis[j / 16] |= static_cast<uint32_t>(norm->axis[j]) << 2 * (j % 16);
  }
  if ((status = check_session(session)) != AFFON_ROCM_OK ||
      (status = check_output(d->output, d->query, *cache, *batch, p.batch, op,
                             {rows_of_view(d->key), rows_of_view(d->value), words(d->positions, q.axes * rows),
                              words(d->rotary, d->rotary_rows * d->rotary_dim), weights[0], weights[1]})) != AFFON_ROCM_OK)
    return status;
  const hipError_t e = affon::append_norm_launch(q, session->stream);
  if (e != hipSuccess) return hip_fail(e, op);
  return AFFON_ROCM_OK;
}

int affon_rocm_tree_attention(affon_rocm_session* session, const affon_rocm_kv_cache* cache,
                              const affon_rocm_draft_batch* batch, const affon_rocm_attention_desc* d) {
  clear_error();
  const char* op = "tree_attention";
  if (d == nullptr) return fail(AFFON_ROCM_INVALID_SHAPE, "%s descriptor is null", op);
  affon::AttentionProblem p{};
  int status = check_attention(cache, batch, d->query, d->mask, d->scale, d->layer, d->output, d->output_bytes, op, &p);
  if (status != AFFON_ROCM_OK) return status;
  p.out = static_cast<uint8_t*>(d->output);
  if ((status = check_session(session)) != AFFON_ROCM_OK ||
      (status = check_output(d->output, d->query, *cache, *batch, p.batch, op, {rows_of_view(d->mask)})) != AFFON_ROCM_OK)
    return status;
  affon::Launch launch;
  launch.stream = session->stream;
  launch.workspace = session->workspace;
  const hipError_t e = affon::attention_launch(p, launch);
  if (e != hipSuccess) return hip_fail(e, op);
  return AFFON_ROCM_OK;
}

int affon_rocm_shared_attention(affon_rocm_session* session, const affon_rocm_kv_cache* cache,
                                const affon_rocm_draft_batch* batch, const affon_rocm_attention_desc* d,
                                const uint32_t* shared, int64_t groups) {
  clear_error();
  const char* op = "shared_attention";
  if (d == nullptr) return fail(AFFON_ROCM_INVALID_SHAPE, "%s descriptor is null", op);
  affon::AttentionProblem p{};
  int status = check_attention(cache, batch, d->query, d->mask, d->scale, d->layer, d->output, d->output_bytes, op, &p);
  if (status != AFFON_ROCM_OK) return status;
  p.out = static_cast<uint8_t*>(d->output);
  if (shared == nullptr || !aligned(shared, 4) || groups <= 0 || p.batch.sequences % groups != 0)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires u32 numbers of shared tokens, of groups of equal size", op);
  if ((status = check_session(session)) != AFFON_ROCM_OK ||
      (status = check_output(d->output, d->query, *cache, *batch, p.batch, op,
                             {rows_of_view(d->mask), words(shared, groups)})) != AFFON_ROCM_OK)
    return status;
  affon::Launch launch;
  launch.stream = session->stream;
  launch.workspace = session->workspace;
  const hipError_t e = affon::shared_attention_launch(p, shared, static_cast<int>(groups), launch);
  if (e != hipSuccess) return hip_fail(e, op);
  return AFFON_ROCM_OK;
}

int affon_rocm_token_weights(affon_rocm_session* session, const affon_rocm_kv_cache* cache,
                             const affon_rocm_draft_batch* batch, float* weights, size_t weights_bytes) {
  clear_error();
  const char* op = "token_weights";
  affon::PagedCache c{};
  affon::DraftBatch b{};
  int status = check_cache(cache, -1, op, &c);
  if (status != AFFON_ROCM_OK || (status = check_batch(batch, c, op, &b)) != AFFON_ROCM_OK) return status;
  affon::Rows to;
  if ((status = check_weights(*cache, b, weights, weights_bytes, op, &to)) != AFFON_ROCM_OK ||
      (status = check_session(session)) != AFFON_ROCM_OK)
    return status;
  if (meets(to, *cache, *batch, b, {})) return fail(AFFON_ROCM_INVALID_SHAPE, "%s weights overlap an operand", op);
  const int64_t count = static_cast<int64_t>(c.layers) * b.sequences * c.kv_heads * static_cast<int64_t>(b.capacity);
  const hipError_t e = affon::clear_weights_launch(weights, count, session->stream);
  if (e != hipSuccess) return hip_fail(e, op);
  return AFFON_ROCM_OK;
}

int affon_rocm_attention_weights(affon_rocm_session* session, const affon_rocm_kv_cache* cache,
                                 const affon_rocm_draft_batch* batch, const affon_rocm_weights_desc* d) {
  clear_error();
  const char* op = "attention_weights";
  if (d == nullptr) return fail(AFFON_ROCM_INVALID_SHAPE, "%s descriptor is null", op);
  affon::AttentionProblem p{};
  int status = check_attention(cache, batch, d->query, d->mask, d->scale, d->layer, nullptr, 0, op, &p, false);
  if (status != AFFON_ROCM_OK) return status;
  affon::Rows weights;
  if ((status = check_weights(*cache, p.batch, d->weights, d->weights_bytes, op, &weights)) != AFFON_ROCM_OK ||
      (status = check_session(session)) != AFFON_ROCM_OK)
    return status;
  if (meets(weights, *cache, *batch, p.batch, {rows_of_view(d->query), rows_of_view(d->mask)}))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s weights overlap an operand", op);
  float* layer = d->weights + d->layer * p.batch.sequences * p.cache.kv_heads * static_cast<int64_t>(p.batch.capacity);
  affon::Launch launch;
  launch.stream = session->stream;
  launch.workspace = session->workspace;
  const hipError_t e = affon::attention_weights_launch(p, layer, launch);
  if (e != hipSuccess) return workspace_fail(e, op);
  return AFFON_ROCM_OK;
}

int affon_rocm_cache_evict(affon_rocm_session* session, const affon_rocm_kv_cache* cache,
                           const affon_rocm_draft_batch* batch, const float* weights, float* out, size_t bytes,
                           const uint32_t* keep, const uint32_t* recent) {
  clear_error();
  const char* op = "cache_evict";
  affon::PagedCache c{};
  affon::DraftBatch b{};
  int status = check_cache(cache, -1, op, &c);
  if (status != AFFON_ROCM_OK || (status = check_batch(batch, c, op, &b)) != AFFON_ROCM_OK) return status;
  affon::Rows in, to;
  if ((status = check_weights(*cache, b, weights, bytes, op, &in)) != AFFON_ROCM_OK ||
      (status = check_weights(*cache, b, out, bytes, op, &to)) != AFFON_ROCM_OK)
    return status;
  if (keep == nullptr || recent == nullptr || !aligned(keep, 4) || !aligned(recent, 4))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires u32 numbers of tokens to keep, and of recent ones", op);
  if ((status = check_session(session)) != AFFON_ROCM_OK) return status;
  const affon::Rows k = words(keep, b.sequences), r = words(recent, b.sequences);
  if ((weights != out && affon::rows_meet(in, to)) || meets(to, *cache, *batch, b, {k, r}))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s output overlaps an operand that it is not", op);
  affon::Launch launch;
  launch.stream = session->stream;
  launch.workspace = session->workspace;
  const hipError_t e = affon::evict_launch(c, b, weights, out, keep, recent, launch);
  if (e != hipSuccess) return workspace_fail(e, op);
  return AFFON_ROCM_OK;
}

int affon_rocm_cache_commit(affon_rocm_session* session, const affon_rocm_kv_cache* cache,
                            const affon_rocm_draft_batch* batch, const affon_rocm_view* path,
                            const uint32_t* accepted) {
  clear_error();
  const char* op = "cache_commit";
  affon::PagedCache c{};
  affon::DraftBatch b{};
  int status = check_commit(cache, batch, path, accepted, op, &c, &b);
  if (status != AFFON_ROCM_OK) return status;
  if ((status = check_session(session)) != AFFON_ROCM_OK) return status;
  const hipError_t e = affon::commit_launch(c, b, reinterpret_cast<const uint32_t*>(origin(*path)), path->stride[0],
                                            static_cast<int>(path->shape[1]), accepted, session->stream);
  if (e != hipSuccess) return hip_fail(e, op);
  return AFFON_ROCM_OK;
}

int affon_rocm_weights_commit(affon_rocm_session* session, const affon_rocm_kv_cache* cache,
                              const affon_rocm_draft_batch* batch, const affon_rocm_view* path,
                              const uint32_t* accepted, float* weights, size_t weights_bytes) {
  clear_error();
  const char* op = "cache_commit";
  affon::PagedCache c{};
  affon::DraftBatch b{};
  int status = check_commit(cache, batch, path, accepted, op, &c, &b);
  if (status != AFFON_ROCM_OK) return status;
  affon::Rows to;
  if ((status = check_weights(*cache, b, weights, weights_bytes, op, &to)) != AFFON_ROCM_OK ||
      (status = check_session(session)) != AFFON_ROCM_OK)
    return status;
  if (meets(to, *cache, *batch, b, {rows_of_view(*path), words(accepted, b.sequences)}))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s weights overlap an operand", op);
  const hipError_t e = affon::commit_weights_launch(b, c.layers, c.kv_heads, weights,
                                                    reinterpret_cast<const uint32_t*>(origin(*path)), path->stride[0],
                                                    static_cast<int>(path->shape[1]), accepted, session->stream);
  if (e != hipSuccess) return hip_fail(e, op);
  return AFFON_ROCM_OK;
}

int affon_rocm_residual_norm(affon_rocm_session* session, const affon_rocm_residual_norm_desc* d) {
  clear_error();
  const char* op = "residual_norm";
  if (d == nullptr) return fail(AFFON_ROCM_INVALID_SHAPE, "%s descriptor is null", op);
  for (int dtype : {d->stream_dtype, d->update_dtype, d->gate_dtype, d->weight_dtype, d->normalized_dtype})
    if (!is_float_dtype(dtype)) return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires f32 or bf16 tensors", op);
  uint64_t count = 0;
  if (!extent({d->rows, d->cols}, &count) || d->rows > kMaxInt || d->cols > (int64_t(1) << 28))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s requires a non-empty rank-two tensor of at most 2^40 values", op);
  if (d->stream == nullptr || d->normalized == nullptr || (d->update != nullptr && d->stream_out == nullptr))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s buffer is null", op);
  if (d->update == nullptr && (d->gate != nullptr || d->post_norm != 0))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s without an update takes no gate and no post_norm", op);
  if (d->post_norm == 0 && d->post_weight != nullptr)
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s post_weight needs post_norm", op);
  // Without an update a stream that is its own output is left alone, whatever its stride.
  const bool kept = d->update == nullptr && d->stream_out == d->stream &&
                    (d->rows == 1 || d->stream_out_stride == d->stream_stride);
  affon_rocm_residual_norm_desc run = *d;
  if (kept) run.stream_out = nullptr;
  const struct {
    const void* data;
    int dtype;
    int64_t stride, least;
  } operands[] = {{d->stream, d->stream_dtype, d->stream_stride, 0},
                  {d->update, d->update_dtype, d->update_stride, 0},
                  {d->gate, d->gate_dtype, d->gate_stride, 0},
                  {d->post_weight, d->weight_dtype, 0, 0},
                  {d->weight, d->weight_dtype, 0, 0},
                  {run.stream_out, d->stream_dtype, d->stream_out_stride, d->cols},
                  {d->normalized, d->normalized_dtype, d->normalized_stride, d->cols}};
  for (const auto& o : operands) {
    if (o.data == nullptr) continue;
    if (!aligned(o.data, element_size(o.dtype)))
      return fail(AFFON_ROCM_INVALID_SHAPE, "%s buffer is not element aligned", op);
    // Rows of an output do not overlap.
    if (o.stride < 0 || (d->rows > 1 && o.stride < o.least) || o.stride > (int64_t(1) << 40) / d->rows)
      return fail(AFFON_ROCM_INVALID_SHAPE, "%s has an invalid row stride", op);
  }
  if (!(d->epsilon > 0.0f) || d->epsilon == std::numeric_limits<float>::infinity())
    return fail(AFFON_ROCM_INVALID_SHAPE, "invalid residual_norm options: epsilon must be finite and positive");
  if (!(d->scale - d->scale == 0.0f)) return fail(AFFON_ROCM_INVALID_SHAPE, "invalid residual_norm options: scale must be finite");
  int status = check_session(session);
  if (status != AFFON_ROCM_OK) return status;

  // An output may be the stream, update or gate itself: a thread reads its
  // values of a row before it writes them. What overlaps in another way would
  // be read by threads and rows after others have written there.
  auto rows = [&](const void* data, int dtype, int64_t stride) {
    const int size = element_size(dtype);
    return affon::rows_of(data, d->rows, d->cols * size, stride * size);
  };
  const affon::Rows stream = rows(d->stream, d->stream_dtype, d->stream_stride);
  const affon::Rows stream_out = rows(run.stream_out, d->stream_dtype, d->stream_out_stride);
  const affon::Rows normalized = rows(d->normalized, d->normalized_dtype, d->normalized_stride);
  if (affon::rows_meet(kept ? stream : stream_out, normalized))
    return fail(AFFON_ROCM_INVALID_SHAPE, "%s outputs overlap", op);
  const affon::Rows inputs[] = {stream, rows(d->update, d->update_dtype, d->update_stride),
                                rows(d->gate, d->gate_dtype, d->gate_stride),
                                rows(d->post_weight, d->weight_dtype, 0), rows(d->weight, d->weight_dtype, 0)};
  for (const auto& in : inputs)
    for (const auto& out : {stream_out, normalized})
      if (affon::rows_meet(in, out) && !affon::same_rows(in, out))
        return fail(AFFON_ROCM_INVALID_SHAPE, "%s output overlaps an operand that it is not", op);
  const hipError_t e = affon::residual_norm_launch(run, session->stream);
  if (e != hipSuccess) return hip_fail(e, op);
  return AFFON_ROCM_OK;
}

// ---- host-pointer drop-in for compute_core_run_quantized_matmul_f32 ----

namespace {

std::mutex g_default_mutex;
affon_rocm_session* g_default_session = nullptr;

struct DeviceBuffer {
  affon_rocm_session* session;
  void* ptr = nullptr;
  explicit DeviceBuffer(affon_rocm_session* s) : session(s) {}
  // Not affon_rocm_free, which clears the message of the step that failed.
  ~DeviceBuffer() {
    if (ptr == nullptr) return;
    try {
      hipError_t e = hipSetDevice(session->device);
      (void)session->memory->free(ptr, &e);
    } catch (const std::exception&) {  // the block then goes when the session ends
    }
  }
};

}  // namespace

int compute_core_run_quantized_matmul_f32(const float* activation, size_t activation_count, const uint32_t* weights,
                                          size_t weight_count, const float* scales, size_t scale_count,
                                          const float* biases, size_t bias_count, float* output, size_t output_count,
                                          size_t rows, size_t depth, size_t columns, size_t bits,
                                          size_t group_size) {
  clear_error();
  // compute_core_cyna.zig:1012-1022, in the same order.
  if (rows == 0 || depth == 0 || columns == 0 || group_size == 0 || (bits != 2 && bits != 4 && bits != 8))
    return fail(AFFON_ROCM_INVALID_SHAPE, "invalid quantized matmul shape");
  const size_t per_word = 32 / bits;
  if (depth % per_word != 0 || depth % group_size != 0)
    return fail(AFFON_ROCM_INVALID_SHAPE, "depth must divide into complete words and groups");
  uint64_t a_count = 0, w_count = 0, g_count = 0, o_count = 0;
  if (!mul_ok(rows, depth, &a_count) || !mul_ok(columns, depth / per_word, &w_count) ||
      !mul_ok(columns, depth / group_size, &g_count) || !mul_ok(rows, columns, &o_count))
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantized matmul counts overflow");
  if (activation_count != a_count || weight_count != w_count || scale_count != g_count || bias_count != g_count ||
      output_count != o_count)
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantized matmul buffer counts do not match the shape");
  if (activation == nullptr || weights == nullptr || scales == nullptr || biases == nullptr || output == nullptr)
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantized matmul buffer is null");
  uint64_t a_bytes, w_bytes, g_bytes, o_bytes;
  if (!mul_ok(a_count, 4, &a_bytes) || !mul_ok(w_count, 4, &w_bytes) || !mul_ok(g_count, 4, &g_bytes) ||
      !mul_ok(o_count, 4, &o_bytes))
    return fail(AFFON_ROCM_INVALID_SHAPE, "quantized matmul byte counts overflow");

  std::lock_guard<std::mutex> lock(g_default_mutex);
  if (g_default_session == nullptr) {
    int status = affon_rocm_session_create(0, &g_default_session);
    if (status != AFFON_ROCM_OK) {
      g_default_session = nullptr;
      return AFFON_ROCM_CORE_FAILURE;
    }
  }
  affon_rocm_session* s = g_default_session;
  DeviceBuffer dx(s), dw(s), ds(s), db(s), dout(s);
  int status;
  if ((status = affon_rocm_alloc(s, a_bytes, &dx.ptr)) != AFFON_ROCM_OK ||
      (status = affon_rocm_alloc(s, w_bytes, &dw.ptr)) != AFFON_ROCM_OK ||
      (status = affon_rocm_alloc(s, g_bytes, &ds.ptr)) != AFFON_ROCM_OK ||
      (status = affon_rocm_alloc(s, g_bytes, &db.ptr)) != AFFON_ROCM_OK ||
      (status = affon_rocm_alloc(s, o_bytes, &dout.ptr)) != AFFON_ROCM_OK ||
      (status = affon_rocm_memcpy_h2d(s, dx.ptr, activation, a_bytes)) != AFFON_ROCM_OK ||
      (status = affon_rocm_memcpy_h2d(s, dw.ptr, weights, w_bytes)) != AFFON_ROCM_OK ||
      (status = affon_rocm_memcpy_h2d(s, ds.ptr, scales, g_bytes)) != AFFON_ROCM_OK ||
      (status = affon_rocm_memcpy_h2d(s, db.ptr, biases, g_bytes)) != AFFON_ROCM_OK)
    return AFFON_ROCM_CORE_FAILURE;
  const int64_t K = static_cast<int64_t>(depth), N = static_cast<int64_t>(columns), M = static_cast<int64_t>(rows);
  const int64_t KW = K / static_cast<int64_t>(per_word), G = K / static_cast<int64_t>(group_size);
  affon_rocm_qmm_desc d{};
  d.input = {dx.ptr, a_bytes, 0, {M, K}, {K, 1}, AFFON_ROCM_F32};
  d.packed = {dw.ptr, w_bytes, 0, {N, KW}, {KW, 1}, AFFON_ROCM_U32};
  d.scales = {ds.ptr, g_bytes, 0, {N, G}, {G, 1}, AFFON_ROCM_F32};
  d.biases = {db.ptr, g_bytes, 0, {N, G}, {G, 1}, AFFON_ROCM_F32};
  d.output = static_cast<float*>(dout.ptr);
  d.output_bytes = o_bytes;
  d.bits = static_cast<uint32_t>(bits);
  d.group_size = static_cast<uint32_t>(group_size);
  d.implementation = AFFON_ROCM_IMPL_AUTO;
  d.numerical_policy = AFFON_ROCM_BACKEND_EQUIVALENT;
  if ((status = affon_rocm_quantized_matmul(s, &d)) != AFFON_ROCM_OK) return status == 1 ? 1 : AFFON_ROCM_CORE_FAILURE;
  if ((status = affon_rocm_memcpy_d2h(s, output, dout.ptr, o_bytes)) != AFFON_ROCM_OK) return AFFON_ROCM_CORE_FAILURE;
  return AFFON_ROCM_OK;
}

}  // extern "C"
