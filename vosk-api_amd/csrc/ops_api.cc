// C entry points of the 8-bit operators (include/vosk_amd_ops.h): argument
// checks, the device guard, the launch.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>
#include <numeric>

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
    if (e == hipSuccess) return;
    (void)hipGetLastError();  // told here: the next launch's check, whoever's, does not find it
    throw Fatal(std::string("HIP error ") + hipGetErrorString(e));
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
// rows * ld * bytes < 2^31, of rows >= 0 and ld >= 1 of any size
bool Below31Bits(long long rows, long long ld, unsigned bytes) { return rows == 0 || ld <= ((1ll << 31) - 1) / bytes / rows; }
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
  Want((a.m == 1 && !a.from) || a.ldx >= a.k, "quantize_rows: rows of x overlap");
  Want(a.xrows >= 0, "quantize_rows: bad number of rows");
  Want(Aligned(a.x, Bytes(a.type)), "quantize_rows: x is not aligned to its elements");
  Want(Aligned(a.codes, 16) && a.ldc % 16 == 0, "quantize_rows: code rows have to be 16-byte aligned");
  Want(a.ldc >= Int8Padded(a.k), "quantize_rows: code rows are shorter than vamd_op_code_bytes(k)");
  Want(a.cache_rows >= (a.rows ? 0 : a.m), "quantize_rows: fewer code rows than rows");
}

// Whether two matrices of rows x n elements share a byte: their spans do, and
// not as different columns of common rows (in steps of both strides' common
// divisor each has the columns of one row).
struct Extent {
  const void* p;
  long long rows, ld, bytes;  // ld: bytes from row to row; bytes: of a row
};
bool Overlap(const Extent& a, const Extent& b) {
  if (a.rows <= 0 || b.rows <= 0) return false;
  const uintptr_t pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
  if (pa + (uintptr_t)((a.rows - 1) * a.ld + a.bytes) <= pb || pb + (uintptr_t)((b.rows - 1) * b.ld + b.bytes) <= pa) return false;
  const long long g = std::gcd(a.rows > 1 ? a.ld : 0, b.rows > 1 ? b.ld : 0);
  if (g == 0) return true;
  const long long d = pb >= pa ? (long long)((pb - pa) % (uintptr_t)g) : (g - (long long)((pa - pb) % (uintptr_t)g)) % g;  // b's column
  return d < a.bytes || d + b.bytes > g;
}

alignas(16) char kNoWorkspace[16];

void CheckLinear(const LinearInt8& a) {
  Want(a.taps >= 1 && a.taps <= kMaxTaps, "linear_int8: 1 to 16 taps");
  Want(FloatTypeOk(a.out_type), "linear_int8: unknown output type");
  Want(std::isfinite(a.res_scale), "linear_int8: residual_scale has to be finite");
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
  Want(!a.rows || a.m == 1 || a.ldrows >= a.taps, "linear_int8: rows of the row map overlap");
  Want(a.ldo >= a.n || (a.m == 1 && !a.out_to), "linear_int8: output rows overlap");
  Want(a.out_rows >= 0 && a.res_rows >= 0, "linear_int8: bad sizes");
  Want(!a.out_to || Below31Bits(a.out_rows, a.ldo, Bytes(a.out_type)),
       "linear_int8: out has to be below 2^31 bytes where out_to maps its rows");
  Want(a.ldo <= kInt8MaxStride || (a.m == 1 && !a.out_to), "linear_int8: rows of out may be 2^23 elements apart at most");
  Want(Aligned(a.out, Bytes(a.out_type)), "linear_int8: out is not aligned to its elements");
  if (a.residual) {
    Want(FloatTypeOk(a.res_type), "linear_int8: unknown residual type");
    Want(a.ldr >= a.n || (a.m == 1 && !a.res_from), "linear_int8: residual rows overlap");
    Want(!a.res_from || Below31Bits(a.res_rows, a.ldr, Bytes(a.res_type)),
         "linear_int8: residual has to be below 2^31 bytes where res_from maps its rows");
    Want(a.ldr <= kInt8MaxStride || (a.m == 1 && !a.res_from), "linear_int8: rows of residual may be 2^23 elements apart at most");
    Want(Aligned(a.residual, Bytes(a.res_type)), "linear_int8: residual is not aligned to its elements");
    // in place, a lane reads the elements that it writes itself: of the same row, whatever maps it
    const bool same_rows = a.out_to == a.res_from && (!a.out_to || a.m == 1 || a.ldout_to == a.ldres_from);
    const bool in_place = a.out == a.residual && a.out_type == a.res_type && same_rows &&
                          (a.ldo == a.ldr || (a.m == 1 && !a.out_to));
    const long long so = Bytes(a.out_type), sr = Bytes(a.res_type);
    Want(in_place || !Overlap({a.out, a.out_rows, a.ldo * so, a.n * so}, {a.residual, a.res_rows, a.ldr * sr, a.n * sr}),
         "linear_int8: out overlaps residual without being it, row by row through the same map");
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

int vamd_op_quantize_rows(int device, void* stream, const VamdQuantizeRows* p) {
  return Guarded([&] {
    Want(p != nullptr, "quantize_rows: null pointer");
    const QuantizeRows a{p->x, p->type, p->m, p->k, p->ldx, p->rows, p->ldrows, p->from, p->ldfrom,
                         p->from ? p->x_rows : p->m, p->count, p->cache_rows, (int8_t*)p->codes, p->ldc, p->scales};
    CheckRows(a);
    if (a.m == 0) return;
    OnDevice guard(device);
    LaunchQuantizeRows(a, (hipStream_t)stream);
    OnDevice::Check(hipGetLastError());
  });
}

int vamd_op_frame_map(int device, void* stream, const VamdFrameMap* p) {
  return Guarded([&] {
    Want(p != nullptr, "frame_map: null pointer");
    Want(p->streams >= 0 && p->cap >= 0 && p->cap <= INT_MAX, "frame_map: bad sizes");
    Want(p->pages >= 1 && p->page >= 1 && (long long)p->pages * p->page <= INT_MAX, "frame_map: bad pages");
    Want(p->taps >= 1 && p->taps <= kMaxTaps, "frame_map: 1 to 16 offsets");
    Want(p->step >= 1, "frame_map: step has to be at least 1");
    Want(p->starts != nullptr, "frame_map: null pointer");
    Want(p->streams == 0 || (p->lengths && p->first && p->table), "frame_map: null pointer");
    Want(p->streams <= 1 || p->ldt >= p->pages, "frame_map: table rows overlap");
    Want(p->cap == 0 || p->rows, "frame_map: null pointer");
    Want(p->page_stride >= 0 && p->frame_stride >= 0, "frame_map: bad strides");
    FrameMap a{};
    a.lengths = p->lengths;
    a.first = p->first;
    a.streams = p->streams;
    a.table = p->table;
    a.ldt = p->ldt;
    a.pages = p->pages;
    a.page = p->page;
    a.page_stride = p->page_stride;
    a.frame_stride = p->frame_stride;
    a.taps = p->taps;
    a.step = p->step;
    a.clamp = p->clamp ? 1 : 0;
    a.low = p->low;
    a.high = p->high;
    a.starts = p->starts;
    a.rows = p->rows;
    a.cap = p->cap;
    SetOffsets(&a, p->offsets);
    OnDevice guard(device);
    LaunchFrameMap(a, (hipStream_t)stream);
    OnDevice::Check(hipGetLastError());
  });
}

int vamd_op_linear_int8(int device, void* stream, const VamdLinearInt8* p) {
  return Guarded([&] {
    Want(p != nullptr, "linear_int8: null pointer");
    Want(p->m >= 0 && p->n >= 0 && p->m <= kInt8MaxRows && p->n <= kInt8MaxCols, "linear_int8: bad sizes");
    Want(p->k >= 1 && p->k <= kInt8MaxK, "linear_int8: k has to be in [1, 131072]");
    LinearInt8 a{(const int8_t*)p->codes, p->lda, p->scale, p->cache_rows, p->rows, p->ldrows, p->taps, p->count,
                 (const int8_t*)p->w, p->ldw, p->wscale, p->m, p->n, p->k, p->bias, p->gain, p->shift,
                 p->residual, p->ldr, p->residual_type, p->residual_scale, p->relu ? 1 : 0, p->out, p->ldo, p->out_type,
                 p->out_to, p->ldout_to, p->out_to ? p->out_rows : p->m, p->res_from, p->ldres_from,
                 p->res_from ? p->res_rows : p->m};
    QuantizeRows q{};
    if (p->x) {
      Want(!p->codes && !p->scale, "linear_int8: x comes without codes and scale");
      Want(p->taps >= 1 && p->taps <= kMaxTaps, "linear_int8: 1 to 16 taps");
      Want(!p->rows || (p->cache_rows >= 1 && p->cache_rows <= kInt8MaxRows), "linear_int8: bad number of rows of x");
      const int kb = Int8Padded(p->k);
      a.lda = kb;
      a.arows = p->rows ? p->cache_rows : p->m;
      // (without a workspace the checks below still want addresses)
      a.a = (const int8_t*)(LinearFloatFused(p->m, kb, p->taps) ? kNoWorkspace : p->workspace);
      a.sa = (const float*)(a.a + (LinearFloatFused(p->m, kb, p->taps) ? 0 : a.arows * kb));
      q = QuantizeRows{p->x, p->x_type, a.arows, p->k, p->ldx, nullptr, 0, nullptr, 0, a.arows,
                       p->rows ? nullptr : p->count, a.arows, (int8_t*)a.a, kb, (float*)a.sa};
      if (p->m && p->n) CheckRows(q);
    }
    CheckLinear(a);
    if (a.m == 0 || a.n == 0) return;
    a.k = Int8Padded(a.k);
    if (a.m == 1 && !a.out_to) a.ldo = a.n;  // one row: any stride was right
    if (a.m == 1 && !a.res_from) a.ldr = a.n;
    OnDevice guard(device);
    if (p->x) LaunchLinearFloat(a, q, (hipStream_t)stream);
    else LaunchLinearInt8(a, (hipStream_t)stream);
    OnDevice::Check(hipGetLastError());
  });
}

long long vamd_op_linear_workspace(int m, int n, int k, int taps, long long x_rows) {
  if (m < 0 || m > kInt8MaxRows || n < 0 || n > kInt8MaxCols || k < 1 || k > kInt8MaxK || taps < 1 || taps > kMaxTaps ||
      x_rows < 0 || x_rows > kInt8MaxRows) {
    SetLastError("linear_int8: bad sizes");
    return -1;
  }
  if (m == 0 || n == 0 || LinearFloatFused(m, Int8Padded(k), taps)) return 0;
  return x_rows * Int8Padded(k) + 4ll * x_rows;
}

}  // extern "C"
