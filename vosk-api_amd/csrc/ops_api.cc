// C entry points of the 8-bit operators (include/vosk_amd_ops.h): argument
// checks, the device guard, the launch.
#include <hip/hip_runtime.h>

#include <climits>

#include "common.h"
#include "int8_ops.h"
#include "../../include/vosk_amd_ops.h"

using namespace vamd;

namespace {

// The calling thread's device is put back when the call returns.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    Check(hipGetDevice(&before_));
    if (device != before_) {
      Check(hipSetDevice(device));
      changed_ = true;
    }
  }
  ~OnDevice() {
    if (changed_) (void)hipSetDevice(before_);
  }
  static void Check(hipError_t e) {
    if (e != hipSuccess) throw Fatal(std::string("HIP error ") + hipGetErrorString(e));
  }

 private:
  int before_ = 0;
  bool changed_ = false;
};

// A refusal says why and logs nothing: the caller has the message.
void Want(bool ok, const char* what) {
  if (!ok) throw Fatal(what);
}

bool Aligned(const void* p, unsigned n) { return ((uintptr_t)p) % n == 0; }
bool FloatTypeOk(int t) { return t == kFloat32 || t == kFloat16 || t == kBFloat16; }
unsigned Bytes(int t) { return t == kFloat32 ? 4 : 2; }

template <class F>
int Guarded(F f) {
  try {
    f();
    return 0;
  } catch (const std::exception& e) {
    SetLastError(e.what());
  } catch (...) {
    SetLastError("unknown exception");
  }
  return -1;
}

void CheckRows(const QuantizeRows& a) {
  Want(FloatTypeOk(a.type), "quantize_rows: unknown element type");
  Want(a.m >= 0 && a.m <= INT_MAX, "quantize_rows: bad number of rows");
  Want(a.k >= 1 && a.k <= kInt8MaxK, "quantize_rows: k has to be in [1, 131072]");
  if (a.m == 0) return;
  Want(a.x && a.codes && a.scales, "quantize_rows: null pointer");
  Want(a.m == 1 || a.ldx >= a.k, "quantize_rows: rows of x overlap");
  Want(Aligned(a.x, Bytes(a.type)), "quantize_rows: x is not aligned to its elements");
  Want(Aligned(a.codes, 16) && a.ldc % 16 == 0, "quantize_rows: code rows have to be 16-byte aligned");
  Want(a.ldc >= Int8Padded(a.k), "quantize_rows: code rows are shorter than vamd_op_code_bytes(k)");
  Want(a.cache_rows >= (a.rows ? 0 : a.m), "quantize_rows: fewer code rows than rows");
}

void CheckLinear(const LinearInt8& a) {
  Want(a.m >= 0 && a.n >= 0 && a.m <= kInt8MaxRows && a.n <= kInt8MaxRows, "linear_int8: bad sizes");
  Want(a.k >= 1 && a.k <= kInt8MaxK, "linear_int8: k has to be in [1, 131072]");
  Want(a.taps >= 1 && a.taps <= kMaxTaps, "linear_int8: 1 to 16 taps");
  Want(FloatTypeOk(a.out_type), "linear_int8: unknown output type");
  if (a.m == 0 || a.n == 0) return;
  const long long kb = Int8Padded(a.k);
  Want(a.a && a.sa && a.w && a.sw && a.out, "linear_int8: null pointer");
  Want(Aligned(a.a, 16) && a.lda % 16 == 0 && Aligned(a.w, 16) && a.ldw % 16 == 0,
       "linear_int8: codes and weights have to be 16-byte aligned, row strides multiples of 16");
  Want(a.arows >= 1 && (a.lda >= kb || a.arows == 1), "linear_int8: code rows are shorter than vamd_op_code_bytes(k)");
  Want(a.ldw >= kb * a.taps || a.n == 1, "linear_int8: weight rows are shorter than taps * vamd_op_code_bytes(k)");
  Want(a.rows || a.taps == 1, "linear_int8: more than one tap needs a row map");
  Want(a.rows || a.arows >= a.m, "linear_int8: fewer code rows than output rows");
  Want(!a.gain == !a.shift, "linear_int8: gain and shift go together");
  Want(a.ldo >= a.n || a.m == 1, "linear_int8: output rows overlap");
  Want(Aligned(a.out, Bytes(a.out_type)), "linear_int8: out is not aligned to its elements");
  if (a.residual) {
    Want(FloatTypeOk(a.res_type), "linear_int8: unknown residual type");
    Want(Aligned(a.residual, Bytes(a.res_type)), "linear_int8: residual is not aligned to its elements");
  }
}

}  // namespace

extern "C" {

int vamd_op_code_bytes(int k) {
  if (k < 1 || k > kInt8MaxK) {
    SetLastError("k has to be in [1, 131072]");
    return -1;
  }
  return Int8Padded(k);
}

int vamd_op_quantize_rows(int device, void* stream, const void* x, int type, long long m, int k, long long ldx,
                          const int* rows, const int* count, long long cache_rows, signed char* codes, long long ldc,
                          float* scales) {
  return Guarded([&] {
    const QuantizeRows a{x, type, m, k, ldx, rows, count, cache_rows, (int8_t*)codes, ldc, scales};
    CheckRows(a);
    if (m == 0) return;
    OnDevice guard(device);
    LaunchQuantizeRows(a, (hipStream_t)stream);
    OnDevice::Check(hipGetLastError());
  });
}

int vamd_op_frame_map(int device, void* stream, const int* lengths, const int* first, int streams, const int* table,
                      long long ldt, int pages, int page, const int* offsets, int taps, int step, const int* low,
                      const int* high, int clamp, int* starts, int* rows, long long cap) {
  return Guarded([&] {
    Want(streams >= 0 && cap >= 0 && cap <= INT_MAX, "frame_map: bad sizes");
    Want(pages >= 1 && page >= 1 && (long long)pages * page <= INT_MAX, "frame_map: bad pages");
    Want(taps >= 1 && taps <= kMaxTaps && offsets, "frame_map: 1 to 16 offsets");
    Want(step >= 1, "frame_map: step has to be at least 1");
    Want(starts != nullptr, "frame_map: null pointer");
    Want(streams == 0 || (lengths && first && table), "frame_map: null pointer");
    Want(streams <= 1 || ldt >= pages, "frame_map: table rows overlap");
    Want(cap == 0 || rows, "frame_map: null pointer");
    FrameMap a{lengths, first, streams, table, ldt, pages, page, taps, step, clamp ? 1 : 0,
               low, high, starts, rows, cap, INT_MIN, {}};
    for (int j = 0; j < taps; j++) {
      a.offset[j] = offsets[j];
      if (offsets[j] > a.max_offset) a.max_offset = offsets[j];
    }
    OnDevice guard(device);
    LaunchFrameMap(a, (hipStream_t)stream);
    OnDevice::Check(hipGetLastError());
  });
}

int vamd_op_linear_int8(int device, void* stream, const signed char* codes, long long lda, const float* scale,
                        long long cache_rows, const int* rows, int taps, const int* count, const signed char* w,
                        long long ldw, const float* wscale, int m, int n, int k, const float* bias, int relu,
                        const float* gain, const float* shift, const void* residual, long long ldr, int residual_type,
                        float residual_scale, void* out, long long ldo, int out_type) {
  return Guarded([&] {
    LinearInt8 a{(const int8_t*)codes, lda, scale, cache_rows, rows, taps, count, (const int8_t*)w, ldw, wscale,
                 m, n, k, bias, gain, shift, residual, ldr, residual_type, residual_scale, relu ? 1 : 0,
                 out, ldo, out_type};
    CheckLinear(a);
    if (m == 0 || n == 0) return;
    a.k = Int8Padded(k);
    OnDevice guard(device);
    LaunchLinearInt8(a, (hipStream_t)stream);
    OnDevice::Check(hipGetLastError());
  });
}

long long vamd_op_linear_workspace(int m, int k) {
  if (m < 0 || k < 1 || k > kInt8MaxK) {
    SetLastError("bad sizes");
    return -1;
  }
  return (long long)m * Int8Padded(k) + 4ll * m;
}

int vamd_op_linear_float(int device, void* stream, const void* x, int type, long long ldx, void* workspace,
                         const int* count, const signed char* w, long long ldw, const float* wscale, int m, int n, int k,
                         const float* bias, int relu, const float* gain, const float* shift, const void* residual,
                         long long ldr, int residual_type, float residual_scale, void* out, long long ldo,
                         int out_type) {
  return Guarded([&] {
    Want(k >= 1 && k <= kInt8MaxK, "linear_float: k has to be in [1, 131072]");
    const int kb = Int8Padded(k);
    int8_t* codes = (int8_t*)workspace;
    float* scales = (float*)(codes + (long long)m * kb);
    const QuantizeRows q{x, type, m, k, ldx, nullptr, count, m, codes, kb, scales};
    LinearInt8 a{codes, kb, scales, m, nullptr, 1, count, (const int8_t*)w, ldw, wscale, m, n, k, bias, gain, shift,
                 residual, ldr, residual_type, residual_scale, relu ? 1 : 0, out, ldo, out_type};
    if (m != 0 && n != 0) CheckRows(q);
    CheckLinear(a);
    if (m == 0 || n == 0) return;
    a.k = kb;
    OnDevice guard(device);
    LaunchQuantizeRows(q, (hipStream_t)stream);
    LaunchLinearInt8(a, (hipStream_t)stream);
    OnDevice::Check(hipGetLastError());
  });
}

}  // extern "C"
