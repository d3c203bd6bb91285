// The 8-bit operators (int8_ops.hip): per-row quantisation, row maps of frame
// caches, and the matrix product over 8-bit codes.  Behind the C entry points
// of include/vosk_amd_ops.h and the engine's 8-bit acoustic model.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace vamd {

enum FloatType { kFloat32 = 0, kFloat16 = 1, kBFloat16 = 2 };

constexpr int kMaxTaps = 16;
constexpr int kInt8Pad = 64;         // code rows are a multiple of 64 bytes per tap
constexpr int kInt8MaxK = 1 << 17;   // a tap's sum of 127 * 127 * K stays in 32 bits
constexpr long long kInt8MaxStride = 1 << 23;  // 32 rows of floats in a buffer of 2^30 bytes
constexpr int kInt8MaxRows = 1 << 30, kInt8MaxCols = 1 << 23;  // of one product
inline int Int8Padded(int k) { return (k + kInt8Pad - 1) / kInt8Pad * kInt8Pad; }

// Codes and scales of M rows of k floats:
//   s = fl32(max |x| / 127),  c = x / s rounded half to even (exact quotient)
// A row of zeros gives s = 0, c = 0; a row holding an Inf or a NaN gives
// s = NaN, c = 0, so whatever is computed from it is NaN.  Columns [k,
// padded k) of a code row are zeroed.  rows (optional): row m goes to row
// rows[m] of a cache of `cache_rows` rows; an entry outside it is skipped.
struct QuantizeRows {
  const void* x;
  int type;            // FloatType
  long long m;
  int k;
  long long ldx;       // elements
  const int* rows;
  long long ldrows;    // entries apart
  const int* from;     // row m is row from[m] of x's `xrows`, skipped outside them (nullptr: m)
  long long ldfrom, xrows;
  const int* count;    // device: rows from *count on are skipped (or nullptr)
  long long cache_rows;
  int8_t* codes;
  long long ldc;       // bytes, a multiple of 16
  float* scales;
};
void LaunchQuantizeRows(const QuantizeRows& a, hipStream_t s);

// Division by a number that is fixed for the launch: the high word of a
// product with a rounded reciprocal (Granlund and Montgomery, "Division by
// invariant integers using multiplication", 1994; exact for all 32-bit n).
struct Divider {
  uint32_t d = 1, magic = 1;
  int s1 = 0, s2 = 0;
  Divider() = default;
  explicit Divider(uint32_t by) : d(by) {
    int l = 0;
    while ((1ull << l) < by) l++;
    magic = (uint32_t)(((1ull << 32) * ((1ull << l) - by)) / by + 1);
    s1 = l < 1 ? l : 1;
    s2 = l > 0 ? l - 1 : 0;
  }
  __host__ __device__ uint32_t div(uint32_t n) const {
    const uint32_t t = (uint32_t)(((uint64_t)magic * n) >> 32);
    return (t + ((n - t) >> s1)) >> s2;
  }
  __host__ __device__ uint32_t mod(uint32_t n) const { return n - div(n) * d; }
};

// Which cache rows the output rows of a step read.  Stream r has lengths[r]
// new frames from time first[r] on and gives n_r = ceil(lengths[r] / step)
// output rows, at times first[r] + step * i; output rows are packed stream
// after stream (starts = exclusive sums of n_r, the total last).  Frame t of
// stream r lies in cache row
//   table[r][(t mod ring) / page] * page_stride + (t mod page) * frame_stride,
// ring = pages * page.  Entry (row, j) names the row of frame t + offset[j],
// t limited to [low[r], high[r]] (clamp: the nearest inside, else -1), -1
// where the page is not assigned, the ring cannot hold the frame beside the
// newest that the stream's rows name, or the row's number passes 31 bits.
struct FrameMap {
  const int* lengths;
  const int* first;
  int streams;
  const int* table;    // [streams][pages], rows ldt apart
  long long ldt;
  int pages, page;
  int page_stride, frame_stride;
  int taps, step, clamp;
  const int* low;      // [streams] or nullptr
  const int* high;
  int* starts;         // [streams + 1]
  int* rows;           // [cap][taps]; rows from the total on are left as they were
  long long cap;
  int max_offset;
  int offset[kMaxTaps];
  Divider by_ring, by_page;
  int per_stream;                 // (the engine's: output rows of each stream)
  bool far_offsets;               // an offset past +-2^30
  unsigned offset_at[kMaxTaps];   // offset mod ring, 0 .. ring - 1
};
// Sets the a->taps offsets and what follows from them and from the pages.
void SetOffsets(FrameMap* a, const int* offsets);
void LaunchFrameMap(const FrameMap& a, hipStream_t s);
// n maps, each with rows and starts of its own, in as few launches as they fit.
constexpr int kMapsPerLaunch = 8;
void LaunchFrameMaps(const FrameMap* maps, int n, hipStream_t s);
inline int FrameMapLaunches(int n) { return (n + kMapsPerLaunch - 1) / kMapsPerLaunch; }

// out[m][n] = epi(sw[n] * sum_j sa[r(m,j)] * sum_k a[r(m,j)][k] * w[n][j * K + k])
// with r(m, j) = rows[m][j] (rows == nullptr: m, taps 1); an entry outside
// [0, arows) adds nothing.  The inner sums are exact in 32-bit integers, the
// rest is 32-bit floats in this order:
//   v = sum over j ascending of fma(float(sum_j), sa_j, v)
//   v = v * sw[n];  v = v + bias[n];  v = max(v, 0) (NaN stays);
//   v = v * gain[n] + shift[n];  v = res_scale * residual[m][n] + v
struct LinearInt8 {
  const int8_t* a;
  long long lda;       // bytes, a multiple of 16
  const float* sa;
  long long arows;
  const int* rows;
  long long ldrows;    // entries apart
  int taps;
  const int* count;    // device: output rows from *count on are left as they were (or nullptr)
  const int8_t* w;
  long long ldw;       // bytes, a multiple of 16
  const float* sw;
  int m, n, k;         // k: columns of one tap, a multiple of kInt8Pad
  const float* bias;
  const float* gain;
  const float* shift;
  const void* residual;
  long long ldr;       // elements
  int res_type;
  float res_scale;
  int relu;
  void* out;
  long long ldo;       // elements
  int out_type;
  // Output row m goes to row out_to[m] of out (of out_rows rows; skipped
  // outside them), and residual row m is row res_from[m] (adds nothing outside
  // res_rows); nullptr: m.  Such a matrix is smaller than 2^31 bytes.
  const int* out_to;
  long long ldout_to, out_rows;
  const int* res_from;
  long long ldres_from, res_rows;
};
void LaunchLinearInt8(const LinearInt8& a, hipStream_t s);
// The product of float rows x, gathered through a's row map: x's codes and
// scales (of all its rows) are a's, a workspace that is not used where
// LinearFloatFused: one launch then quantises the rows it reads in LDS, to the
// same codes.
bool LinearFloatFused(int m, int k, int taps);
void LaunchLinearFloat(const LinearInt8& a, const QuantizeRows& x, hipStream_t s);
}  // namespace vamd
