// 8-bit operators (int8_ops.h; gfx950): per-row quantisation, row maps of
// frame caches, the matrix product over 8-bit codes on int8 MFMA.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <climits>

#include "common.h"
#include "int8_ops.h"

namespace vamd {

namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float load_float(const void* p, int type, long long i) {
  if (type == kFloat32) return ((const float*)p)[i];
  if (type == kFloat16) return __half2float(((const __half*)p)[i]);
  return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
}

// round to nearest even; a NaN stays a (quiet) NaN
__device__ __forceinline__ uint16_t to_bf16(float v) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

__device__ __forceinline__ void store_float(void* p, int type, long long i, float v) {
  if (type == kFloat32) ((float*)p)[i] = v;
  else if (type == kFloat16) ((__half*)p)[i] = __float2half(v);
  else ((uint16_t*)p)[i] = to_bf16(v);
}

// x / s rounded half to even, exactly: r = rint(x * (1 / s)) is off by one at
// most; d = x - r * s is exact in 32 bits (a multiple of the smaller of the
// two units in the last place, and no larger than s), so comparing it with
// s / 2 decides.
__device__ __forceinline__ int code_of(float x, float s, float inv) {
  float r = rintf(x * inv);
  const float d = fmaf(-r, s, x), h = 0.5f * s;
  const float ad = fabsf(d);
  if (ad > h || (ad == h && ((int)r & 1))) r += d > 0.0f ? 1.0f : -1.0f;
  r = fminf(fmaxf(r, -127.0f), 127.0f);
  return (int)r;
}

// ---- rows to codes: one wave per row, two passes
template <int TYPE>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeRows a) {
  const int lane = threadIdx.x & 63;
  const long long m = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= a.m || (a.count && m >= *a.count)) return;
  const long long to = a.rows ? a.rows[m] : m;
  if (to < 0 || to >= a.cache_rows) return;
  uint32_t top = 0;
  for (int i = lane; i < a.k; i += 64) {
    const uint32_t u = __float_as_uint(load_float(a.x, TYPE, m * a.ldx + i)) & 0x7fffffffu;
    top = u > top ? u : top;
  }
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t u = __shfl_xor(top, o);
    top = u > top ? u : top;
  }
  const bool fine = top < 0x7f800000u;
  float s = fine ? __uint_as_float(top) / 127.0f : __uint_as_float(0x7fc00000u);
  if (lane == 0) a.scales[to] = s;
  const bool zero = !(s > 0.0f);
  // scales near the end of the range are brought up so that 1 / s is finite
  const float up = s < 0x1p-100f ? 0x1p100f : 1.0f;
  s = zero ? 1.0f : s * up;
  const float inv = 1.0f / s;
  int8_t* c = a.codes + to * a.ldc;
  const int kp = (a.k + kInt8Pad - 1) / kInt8Pad * kInt8Pad;
  for (int i = lane; i < kp; i += 64)
    c[i] = i < a.k && !zero ? (int8_t)code_of(load_float(a.x, TYPE, m * a.ldx + i) * up, s, inv) : (int8_t)0;
}

// ---- row maps
constexpr int kMapThreads = 256;

// exclusive sums of the streams' row counts: one workgroup
__global__ __launch_bounds__(kMapThreads) void frame_starts_kernel(FrameMap a) {
  __shared__ long long part[kMapThreads];
  const int tid = threadIdx.x;
  const int per = (a.streams + kMapThreads - 1) / kMapThreads;
  const int lo = min(tid * per, a.streams), hi = min(lo + per, a.streams);
  long long sum = 0;
  for (int r = lo; r < hi; r++) sum += (max(a.lengths[r], 0) + (long long)a.step - 1) / a.step;
  part[tid] = sum;
  __syncthreads();
  for (int o = 1; o < kMapThreads; o <<= 1) {
    const long long v = tid >= o ? part[tid - o] : 0;
    __syncthreads();
    part[tid] += v;
    __syncthreads();
  }
  long long at = part[tid] - sum;
  for (int r = lo; r < hi; r++) {
    a.starts[r] = (int)min(at, (long long)INT_MAX);
    at += (max(a.lengths[r], 0) + (long long)a.step - 1) / a.step;
  }
  if (tid == kMapThreads - 1) a.starts[a.streams] = (int)min(part[tid], (long long)INT_MAX);
}

__global__ __launch_bounds__(kMapThreads) void frame_map_kernel(FrameMap a) {
  const long long total = a.starts[a.streams];
  const long long rows = min(total, a.cap);
  const int ring = a.pages * a.page;
  for (long long row = (long long)blockIdx.x * kMapThreads + threadIdx.x; row < rows;
       row += (long long)gridDim.x * kMapThreads) {
    int lo = 0, hi = a.streams - 1;  // the last stream whose first row is not after this one
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.starts[mid] <= row) lo = mid;
      else hi = mid - 1;
    }
    const int r = lo;
    const long long n = (max(a.lengths[r], 0) + (long long)a.step - 1) / a.step;
    const long long t0 = a.first[r] + (long long)a.step * (row - a.starts[r]);
    long long newest = a.first[r] + (long long)a.step * (n - 1) + a.max_offset;
    if (a.high) newest = min(newest, (long long)a.high[r]);
    for (int j = 0; j < a.taps; j++) {
      long long t = t0 + a.offset[j];
      if (a.clamp) {
        if (a.low) t = max(t, (long long)a.low[r]);
        if (a.high) t = min(t, (long long)a.high[r]);
      }
      bool held = t > newest - ring && t >= INT_MIN && t <= INT_MAX;
      if (a.low) held = held && t >= a.low[r];
      if (a.high) held = held && t <= a.high[r];
      int to = -1;
      if (held) {
        int at = (int)t % ring;
        if (at < 0) at += ring;
        const int pg = a.table[r * a.ldt + at / a.page];
        if (pg >= 0) to = pg * a.page + at % a.page;
      }
      a.rows[row * a.taps + j] = to;
    }
  }
}

// ---- the product: one wave per 32 x 32 block of the output, operands
// streamed from global memory into v_mfma_i32_32x32x32_i8 (lane half h holds
// 16 bytes of its row / column; the accumulator of lane l is column l & 31,
// rows (i & 3) + 8 * (i >> 2) + 4 * (l >> 5))
__device__ __forceinline__ float finish(const LinearInt8& a, float v, long long m, int n, float sw) {
  v = v * sw;
  if (a.bias) v = v + a.bias[n];
  if (a.relu) v = v < 0.0f ? 0.0f : v;
  if (a.gain) v = v * a.gain[n] + a.shift[n];
  if (a.residual) v = a.res_scale * load_float(a.residual, a.res_type, m * a.ldr + n) + v;
  return v;
}

__global__ __launch_bounds__(64) void linear_int8_kernel(LinearInt8 a) {
  __shared__ float srow[32];
  const int lane = threadIdx.x, r = lane & 31, h = lane >> 5;
  const int m0 = blockIdx.x * 32, n0 = blockIdx.y * 32;
  const int mrows = a.count ? min(a.m, *a.count) : a.m;
  if (m0 >= mrows) return;
  const int n = n0 + r, nn = n < a.n ? n : a.n - 1;
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; i++) v[i] = 0.0f;
  for (int j = 0; j < a.taps; j++) {
    long long row = -1;
    if (m0 + r < mrows) row = a.rows ? a.rows[(long long)(m0 + r) * a.taps + j] : m0 + r;
    const bool there = row >= 0 && row < a.arows;
    if (!there) row = 0;
    __syncthreads();
    if (h == 0) srow[r] = there ? a.sa[row] : 0.0f;
    __syncthreads();
    const int8_t* ap = a.a + row * a.lda + 16 * h;
    const int8_t* wp = a.w + nn * a.ldw + (long long)j * a.k + 16 * h;
    intx16 acc;
#pragma unroll
    for (int i = 0; i < 16; i++) acc[i] = 0;
    for (int k = 0; k < a.k; k += 32) {
      const intx4 x = *reinterpret_cast<const intx4*>(ap + k), w = *reinterpret_cast<const intx4*>(wp + k);
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(x, w, acc, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = fmaf((float)acc[i], srow[(i & 3) + 8 * (i >> 2) + 4 * h], v[i]);
  }
  if (n >= a.n) return;
  const float sw = a.sw[n];
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const int m = m0 + (i & 3) + 8 * (i >> 2) + 4 * h;
    if (m < mrows) store_float(a.out, a.out_type, m * a.ldo + n, finish(a, v[i], m, n, sw));
  }
}

unsigned Blocks(long long n, long long per) {
  const long long b = (n + per - 1) / per;
  if (b > INT_MAX) VAMD_ERR("too many rows for one launch: " << n);
  return (unsigned)b;
}

}  // namespace

void LaunchQuantizeRows(const QuantizeRows& a, hipStream_t s) {
  if (a.m <= 0) return;
  const dim3 grid(Blocks(a.m, 4));
  if (a.type == kFloat32) hipLaunchKernelGGL(quantize_rows_kernel<kFloat32>, grid, dim3(256), 0, s, a);
  else if (a.type == kFloat16) hipLaunchKernelGGL(quantize_rows_kernel<kFloat16>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(quantize_rows_kernel<kBFloat16>, grid, dim3(256), 0, s, a);
}

void LaunchFrameMap(const FrameMap& a, hipStream_t s) {
  hipLaunchKernelGGL(frame_starts_kernel, dim3(1), dim3(kMapThreads), 0, s, a);
  if (a.cap <= 0) return;
  const long long b = (a.cap + kMapThreads - 1) / kMapThreads;
  hipLaunchKernelGGL(frame_map_kernel, dim3((unsigned)(b < 65536 ? b : 65536)), dim3(kMapThreads), 0, s, a);
}

void LaunchLinearInt8(const LinearInt8& a, hipStream_t s) {
  if (a.m <= 0 || a.n <= 0) return;
  const unsigned gy = Blocks(a.n, 32);
  if (gy > 65535) VAMD_ERR("too many columns for one launch: " << a.n);
  hipLaunchKernelGGL(linear_int8_kernel, dim3(Blocks(a.m, 32), gy), dim3(64), 0, s, a);
}

}  // namespace vamd
