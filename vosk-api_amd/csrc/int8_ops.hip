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

__device__ __forceinline__ void store_float(void* p, int type, long long i, float v) {
  if (type == kFloat32) ((float*)p)[i] = v;
  else if (type == kFloat16) ((__half*)p)[i] = __float2half(v);
  else ((__bf16*)p)[i] = (__bf16)v;
}

// x / s rounded half to even, exactly: r = rint(x * (1 / s)) is off by one at
// most; d = x - r * s is exact in 32 bits (a multiple of the smaller of the
// two units in the last place, and no larger than s), so comparing it with
// s / 2 decides.
__device__ __forceinline__ int code_of(float x, float s, float inv) {
  float r = rintf(x * inv);
  const float d = fmaf(-r, s, x), ad = fabsf(d), h = 0.5f * s;
  if (ad >= h) {  // hardly ever
    if (ad > h || ((int)r & 1)) r += d > 0.0f ? 1.0f : -1.0f;
  }
  return (int)__builtin_amdgcn_fmed3f(r, -127.0f, 127.0f);
}

// A row's scale, and what code_of divides by: scales near the end of the
// range are brought up so that 1 / s is finite, x with them.
struct RowScale {
  float scale, s, inv, up;
  bool zero;  // codes 0: a row of zeros, or one that holds an Inf or a NaN
};
__device__ __forceinline__ RowScale row_scale(uint32_t top) {  // top: the largest |x| as bits
  RowScale r;
  r.scale = top < 0x7f800000u ? __uint_as_float(top) / 127.0f : __uint_as_float(0x7fc00000u);
  r.zero = !(r.scale > 0.0f);
  r.up = r.scale < 0x1p-100f ? 0x1p100f : 1.0f;
  r.s = r.zero ? 1.0f : r.scale * r.up;
  r.inv = 1.0f / r.s;
  return r;
}

// A launch has less than 2^32 threads a dimension: more workgroups than kGridX
// go into the next (a multiple of 8, which keeps block_id & 7 the XCD).
constexpr long long kGridX = 1 << 22;
__device__ __forceinline__ long long block_id() { return blockIdx.y * kGridX + blockIdx.x; }
dim3 Grid(long long blocks) {
  if (blocks > INT_MAX) VAMD_ERR("too many workgroups for one launch: " << blocks);
  return blocks <= kGridX ? dim3((unsigned)blocks) : dim3((unsigned)kGridX, (unsigned)((blocks + kGridX - 1) / kGridX));
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t u = __shfl_xor(v, o);
    v = u > v ? u : v;
  }
  return v;
}

// 16 bytes of a row, which may lie at any element; past the row: zeros
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
template <int TYPE>
struct Chunk {
  static constexpr int N = TYPE == kFloat32 ? 4 : 8;  // elements
  uint32_t w[4];
  __device__ __forceinline__ void load(const void* x, long long row0, int e, int k) {
    const char* p = (const char*)x + (row0 + e) * (16 / N);
    if (e + N <= k) {
      __builtin_memcpy(w, p, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) w[i] = 0;
      if (e < k) {  // the row's end: all loads at once, those past it of its last element
        uint32_t v[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
          const char* const q = p + min(i, k - 1 - e) * (16 / N);
          if constexpr (N == 4) __builtin_memcpy(&v[i], q, 4);
          else v[i] = *(const uint16_t*)q;
        }
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = e + i < k ? v[i] : 0u;
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = N == 4 ? v[i] : v[2 * i % N] | v[(2 * i + 1) % N] << 16;
      }
    }
  }
  // the largest |x| so far: 32-bit patterns, or two 16-bit ones at once
  __device__ __forceinline__ uint32_t top(uint32_t t) const {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (N == 4) {
        t = max(t, w[i] & 0x7fffffffu);
      } else {
        t = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, t),
                                                                   __builtin_bit_cast(ushort2v, w[i] & 0x7fff7fffu)));
      }
    }
    return t;
  }
  static __device__ __forceinline__ uint32_t top_bits(uint32_t t) {  // ... as the bits of a 32-bit float
    if constexpr (N == 4) return t;
    t = max(t & 0xffffu, t >> 16);
    if constexpr (TYPE == kBFloat16) return t << 16;
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)t)));
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (TYPE == kFloat32) return __uint_as_float(w[i]);
    if constexpr (TYPE == kBFloat16) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    return __half2float(__ushort_as_half((unsigned short)(w[i / 2] >> (i & 1 ? 16 : 0))));
  }
  // The sum x * (1 / s) + 1.5 * 2^23 is rounded to a whole number, whose low
  // byte is the code; x - code * s, as in code_of, says whether any of the
  // chunk's has to be looked at again.
  __device__ __forceinline__ void store(int8_t* to, const RowScale& r) const {
    uint32_t z[N], out[N / 4];
    constexpr float kWhole = 12582912.0f;
    float off = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float v = value(i), y = fmaf(v, r.inv, kWhole);
      z[i] = __float_as_uint(y);
      off = fmaxf(off, fabsf(fmaf(-(y - kWhole), r.s, v)));
    }
    if (off >= 0.5f * r.s || r.up != 1.0f || r.zero) {
#pragma unroll
      for (int i = 0; i < N; i++) z[i] = r.zero ? 0u : (uint32_t)code_of(value(i) * r.up, r.s, r.inv);
    }
#pragma unroll
    for (int q = 0; q < N / 4; q++)
      out[q] = __builtin_amdgcn_perm(z[4 * q + 1], z[4 * q], 0x0c0c0400u) |
               __builtin_amdgcn_perm(z[4 * q + 3], z[4 * q + 2], 0x04000c0cu);
    __builtin_memcpy(__builtin_assume_aligned(to, N), out, N);
  }
};

// ---- rows to codes
//
// Two passes over a row, its maximum and its codes, and one read of it: TPR
// threads (64 or 256) a row keep it in registers (NV chunks of 16 bytes a
// thread) in between; NV = 0: rows longer than that are read twice.  Bound by
// memory: 13 056 rows of 512 floats (33.5 MB read and written) 6.6 us, 5.0 TB/s,
// what a large copy reaches here; 8 192 rows of 4 096 bf16 (101 MB) 18 us;
// 9 001 rows of 2 047 bf16, whose ends are loaded one by one, 12 to 14 us (55 MB).
// One row of 512: 1.8 us, the launch.
template <int TYPE, int TPR, int NV>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeRows a) {
  constexpr int N = Chunk<TYPE>::N;
  __shared__ uint32_t part[4];
  const int tid = threadIdx.x % TPR;
  const long long m = block_id() * (256 / TPR) + threadIdx.x / TPR;
  long long to = -1;
  long long from = m;
  if (m < a.m && !(a.count && m >= *a.count)) {
    to = a.rows ? a.rows[m * a.ldrows] : m;
    if (a.from) from = a.from[m * a.ldfrom];
  }
  if (to < 0 || to >= a.cache_rows || from < 0 || from >= a.xrows) return;  // the same in all threads of the row
  const int kp = (a.k + kInt8Pad - 1) / kInt8Pad * kInt8Pad;
  const long long row0 = from * a.ldx;
  Chunk<TYPE> c[NV ? NV : 1];
  uint32_t top = 0;
  if (NV) {
#pragma unroll
    for (int i = 0; i < NV; i++) c[i].load(a.x, row0, (i * TPR + tid) * N, a.k);
#pragma unroll
    for (int i = 0; i < NV; i++) top = c[i].top(top);
  } else {
    for (int e = tid * N; e < a.k; e += TPR * N) {
      c[0].load(a.x, row0, e, a.k);
      top = c[0].top(top);
    }
  }
  top = wave_max(Chunk<TYPE>::top_bits(top));
  if (TPR > 64) {  // one row a workgroup
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(part[0], part[1]), max(part[2], part[3]));
  }
  const RowScale r = row_scale(top);
  if (tid == 0) a.scales[to] = r.scale;
  int8_t* const q = a.codes + to * a.ldc;
  if (NV) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int e = (i * TPR + tid) * N;
      if (e < kp) c[i].store(q + e, r);
    }
  } else {
    for (int e = tid * N; e < kp; e += TPR * N) {
      c[0].load(a.x, row0, e, a.k);
      c[0].store(q + e, r);
    }
  }
}

template <int TYPE>
void LaunchQuantize(const QuantizeRows& a, hipStream_t s) {
  constexpr int N = Chunk<TYPE>::N;
  const int kp = Int8Padded(a.k);
  const dim3 rows4 = Grid((a.m + 3) / 4), rows1 = Grid(a.m);
  // A wave a row as long as that takes few registers; of longer rows only where
  // there are so many that they fill the chip (us in a graph, a wave / four
  // waves a row): 512 rows of 1024 floats 3.4 / 3.3, 2048 3.7 / 4.4, 8192 6.8 /
  // 10.2; 2048 rows of 2048 floats 4.6 / 4.8, 4096 6.9 / 8.2; 4096 rows of 2047
  // bf16 8.8 / 8.5, 8192 13.3 / 14.4; 8192 rows of 4096 bf16 22.2 / 18.0.
  const long long many = N == 4 ? 1024 : 4096;
  if (kp <= 64 * N) hipLaunchKernelGGL((quantize_rows_kernel<TYPE, 64, 1>), rows4, dim3(256), 0, s, a);
  else if (kp <= 64 * 2 * N) hipLaunchKernelGGL((quantize_rows_kernel<TYPE, 64, 2>), rows4, dim3(256), 0, s, a);
  else if (kp <= 64 * 4 * N && a.m > many) hipLaunchKernelGGL((quantize_rows_kernel<TYPE, 64, 4>), rows4, dim3(256), 0, s, a);
  else if (TYPE == kFloat32 && kp <= 64 * 8 * N && a.m > 2 * many)
    hipLaunchKernelGGL((quantize_rows_kernel<kFloat32, 64, 8>), rows4, dim3(256), 0, s, a);
  else if (kp <= 256 * 2 * N) hipLaunchKernelGGL((quantize_rows_kernel<TYPE, 256, 2>), rows1, dim3(256), 0, s, a);
  else if (kp <= 256 * 4 * N) hipLaunchKernelGGL((quantize_rows_kernel<TYPE, 256, 4>), rows1, dim3(256), 0, s, a);
  else if (kp <= 256 * 8 * N) hipLaunchKernelGGL((quantize_rows_kernel<TYPE, 256, 8>), rows1, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((quantize_rows_kernel<TYPE, 256, 0>), rows1, dim3(256), 0, s, a);
}

// ---- row maps
//
// A workgroup makes neighbouring output rows of the packed order.  Up to
// kMapStreams streams it sums the streams' row counts itself, in LDS (at most
// 16 KB of lengths out of L2, against a launch of its own for the sums);
// with more, a first launch has written `starts` and the search reads those.
// Bound by latencies one after another (lengths, sums, search, the stream's
// numbers, its pages), not by its bytes: one stream of 51 frames 3.7 to 4.3 us,
// 256 streams 5.2 to 5.8, 4 001 streams and 2 M entries (8 MB) 10.8 to 12.1.
// Larger workgroups sum more streams: 4 001 streams in one of 256 / 512 / 1024
// threads, 400 100 rows of 5 entries 10.4 / 9.2 / 10.2 us, 8 002 rows 8.3 / 7.2 /
// 7.7.
constexpr int kMapThreads = 256, kMapManyThreads = 512, kMapStreams = 4096, kStartsThreads = 1024;

__device__ __forceinline__ unsigned frame_rows(const FrameMap& a, int r) {  // output rows of stream r
  const unsigned n = (unsigned)max(a.lengths[r], 0);
  return a.step == 1 ? n : (n + (unsigned)a.step - 1u) / (unsigned)a.step;
}

// Sums end at 2^32 - 1 instead of wrapping (and at INT_MAX in `starts`).
__device__ __forceinline__ unsigned add_sat(unsigned a, unsigned b) { return __builtin_elementwise_add_sat(a, b); }
__device__ __forceinline__ int saturated(unsigned v) { return (int)min(v, (unsigned)INT_MAX); }

// exclusive sums over the workgroup of THREADS; *total: the sum of all
template <int THREADS>
__device__ __forceinline__ unsigned block_scan(unsigned sum, unsigned* total) {
  __shared__ unsigned part[THREADS / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  unsigned v = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned u = __shfl_up(v, o);
    if (lane >= o) v = add_sat(v, u);
  }
  if (lane == 63) part[wave] = v;
  v = __shfl_up(v, 1);
  if (lane == 0) v = 0;
  __syncthreads();
  unsigned before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; w++) {
    if (w < wave) before = add_sat(before, part[w]);
    all = add_sat(all, part[w]);
  }
  *total = all;
  return add_sat(before, v);
}

// exclusive sums of the streams' row counts: one workgroup
__global__ __launch_bounds__(kStartsThreads) void frame_starts_kernel(FrameMap a) {
  const int tid = threadIdx.x;
  const long long per = (a.streams + kStartsThreads - 1ll) / kStartsThreads;
  const int lo = (int)min(tid * per, (long long)a.streams), hi = (int)min(lo + per, (long long)a.streams);
  unsigned sum = 0, total;
  for (int r = lo; r < hi; r++) sum = add_sat(sum, frame_rows(a, r));
  unsigned at = block_scan<kStartsThreads>(sum, &total);
  for (int r = lo; r < hi; r++) {
    a.starts[r] = saturated(at);
    at = add_sat(at, frame_rows(a, r));
  }
  if (tid == 0) a.starts[a.streams] = saturated(total);
}

// The workgroup sums the streams itself, EACH a thread (0: `starts` is there
// already).  A lane makes ROWS rows, 64 apart, of the ROWS * 64 of its wave,
// their loads in flight together.
template <int THREADS, int EACH, int ROWS>
__device__ __forceinline__ void map_rows(const FrameMap& a) {
  constexpr bool SUM = EACH > 0;
  constexpr int GAP = EACH > 1 ? EACH : 1 << 30;
  // starts; a gap every EACH so that a thread's lie in other banks than its neighbours'
  __shared__ int sums[SUM ? (EACH + 1) * THREADS : 1];
  const int tid = threadIdx.x;
  auto at = [](int r) { return r + r / GAP; };
  unsigned total;
  if constexpr (SUM) {
    constexpr int STRIDE = EACH > 1 ? EACH + 1 : 1;
    unsigned n[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const int r = tid + i * THREADS;
      n[i] = r < a.streams ? frame_rows(a, r) : 0u;
    }
#pragma unroll
    for (int i = 0; i < EACH; i++) sums[at(tid + i * THREADS)] = (int)n[i];
    __syncthreads();
    unsigned sum = 0;
    const bool any = tid * EACH < a.streams;
    if (any) {
#pragma unroll
      for (int i = 0; i < EACH; i++) {
        n[i] = (unsigned)sums[tid * STRIDE + i];
        sum = add_sat(sum, n[i]);
      }
    }
    unsigned v = block_scan<THREADS>(sum, &total);
    if (any) {
#pragma unroll
      for (int i = 0; i < EACH; i++) {
        sums[tid * STRIDE + i] = saturated(v);
        v = add_sat(v, n[i]);
      }
    }
    __syncthreads();
    if (block_id() == 0) {
      for (int r = tid; r < a.streams; r += THREADS) a.starts[r] = sums[at(r)];
      if (tid == 0) a.starts[a.streams] = saturated(total);
    }
  } else {
    total = a.starts[a.streams];
  }
  auto start = [&](int r) { return SUM ? sums[at(r)] : a.starts[r]; };
  // the last stream that begins at or before a row that is the same in all
  // lanes: 64 candidates at a time
  auto wave_stream_of = [&](long long row) {
    long long span = 64;
    while (span < a.streams) span *= 64;
    int base = 0;
    for (span /= 64; span >= 1; span /= 64) {
      const long long r = base + (threadIdx.x & 63) * span;
      base += (int)span * (__popcll(__ballot(r < a.streams && start((int)r) <= row)) - 1);
    }
    return base;
  };
  auto stream_of = [&](int lo, int hi, long long row) {  // the last of them that begins at or before the row
    while (lo < hi) {
      const int mid = (int)(((unsigned)lo + (unsigned)hi + 1u) >> 1);
      if (start(mid) <= row) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };

  const long long rows = min((long long)saturated(total), a.cap);
  const unsigned ring = (unsigned)a.pages * (unsigned)a.page;
  const int lane = tid & 63;
  const long long row0 = (block_id() * THREADS + (tid - lane)) * ROWS;
  if (row0 >= rows) return;
  // the wave's rows are neighbours: those of its first and last row bound the lanes' search
  const int r0 = wave_stream_of(row0), r1 = wave_stream_of(min(row0 + 64 * ROWS, rows) - 1);
  int r[ROWS], low[ROWS], high[ROWS], first[ROWS];
  unsigned n[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; i++) r[i] = stream_of(r0, r1, row0 + i * 64 + lane);
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    first[i] = a.first[r[i]];
    n[i] = frame_rows(a, r[i]);
    low[i] = a.low ? a.low[r[i]] : INT_MIN;
    high[i] = a.high ? a.high[r[i]] : INT_MAX;
  }
  auto mod_ring = [&](int t) {  // 0 .. ring - 1; of a negative t: of -1 - t, from the other end
    const unsigned sign = (unsigned)(t >> 31);
    return (a.by_ring.mod((unsigned)t ^ sign) ^ sign) + (sign & ring);
  };
  long long t0[ROWS];
  int oldest[ROWS];
  bool far = a.far_offsets;  // some time may be outside 32 bits
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    t0[i] = first[i] + (long long)a.step * (row0 + i * 64 + lane - start(r[i]));
    long long newest = first[i] + (long long)a.step * ((long long)n[i] - 1) + a.max_offset;
    if (a.high) newest = min(newest, (long long)high[i]);
    // the first frame that has a row (no limits: INT_MIN and INT_MAX, past which no frame has one either)
    oldest[i] = (int)min(max(newest - ring + 1, (long long)low[i]), (long long)INT_MAX);
    far = far || t0[i] < -(1 << 30) || t0[i] >= (1 << 30);
  }
  far = __any(far);
  // places in the ring of the row's time and of the limits, from which those of the taps follow
  unsigned at0[ROWS], at_low[ROWS], at_high[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    at0[i] = far ? 0u : mod_ring((int)t0[i]);
    at_low[i] = a.clamp && a.low ? mod_ring(low[i]) : 0u;
    at_high[i] = a.clamp && a.high ? mod_ring(high[i]) : 0u;
  }
  // a wave's entries are turned in LDS, so that they go out as whole lines
  extern __shared__ int entries[];  // [waves][ROWS][64][taps]
  int* const turn = entries + (tid >> 6) * ROWS * 64 * a.taps;
  for (int j0 = 0; j0 < a.taps; j0 += 4) {
    int to[ROWS][4];
#pragma unroll
    for (int i = 0; i < ROWS; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        to[i][j] = -1;
        if (j0 + j >= a.taps) break;
        int t;
        unsigned u;
        bool held = true;
        if (!far) {
          t = (int)t0[i] + a.offset[j0 + j];
          u = at0[i] + a.offset_at[j0 + j];
          u = min(u, u - ring);  // (below the ring, the difference wraps and is larger)
        } else {
          const long long wide = t0[i] + a.offset[j0 + j];
          t = (int)min(max(wide, (long long)INT_MIN), (long long)INT_MAX);
          held = t == wide || (a.clamp && ((a.low && wide < low[i]) || (a.high && wide > high[i])));
          u = mod_ring(t);
        }
        if (a.clamp && a.low && t < low[i]) {
          t = low[i];
          u = at_low[i];
        }
        if (a.clamp && a.high && t > high[i]) {
          t = high[i];
          u = at_high[i];
        }
        held = held && t >= oldest[i] && t <= high[i];
        const unsigned q = a.pages == 1 ? 0u : a.by_page.div(u);
        const int pg = held ? a.table[r[i] * a.ldt + q] : -1;
        const uint64_t row = (uint64_t)(unsigned)pg * (unsigned)a.page_stride +
                             (uint64_t)(u - q * (unsigned)a.page) * (unsigned)a.frame_stride;
        if (pg >= 0 && row <= INT_MAX) to[i][j] = (int)row;
      }
#pragma unroll
    for (int i = 0; i < ROWS; i++)
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (j0 + j < a.taps) turn[(i * 64 + lane) * a.taps + j0 + j] = to[i][j];
  }
  const long long left = (rows - row0) * a.taps;
  int* const out = a.rows + row0 * a.taps;
  for (int e = lane; e < ROWS * 64 * a.taps && e < left; e += 64) out[e] = turn[e];
}

template <int THREADS, int EACH, int ROWS>
__global__ __launch_bounds__(THREADS) void frame_map_kernel(FrameMap a) {
  map_rows<THREADS, EACH, ROWS>(a);
}

// several maps in one launch
struct FrameMaps {
  FrameMap map[kMapsPerLaunch];
};
template <int THREADS, int EACH>
__global__ __launch_bounds__(THREADS) void frame_maps_kernel(FrameMaps all) {
  map_rows<THREADS, EACH, 1>(all.map[blockIdx.z]);
}

// ---- the product
//
// Tiles of TM rows x TN columns, WM x WN waves, each wave (TM / WM) x (TN / WN)
// in 32 x 32 blocks of v_mfma_i32_32x32x32_i8 (lane half h holds 16 bytes of
// its row / column; the accumulator of lane l is column l & 31, rows
// (i & 3) + 8 * (i >> 2) + 4 * (l >> 5)).  K goes in parts of 64 bytes, KB
// parts a step: the tile's rows of A (gathered through the row map) and of W go
// straight from global memory into a ring of ST LDS buffers, so ST - 1 steps
// of loads are in flight behind the matrix instructions and one barrier a step
// is enough.  A part's rows are 64 bytes in LDS, their four 16-byte chunks
// permuted by (row >> 2) & 3 (on the global side of the load: LDS takes lane
// after lane), so that the sixteen lanes which a 16-byte-a-lane read serves
// together, four runs of four rows, lie in different banks ((row >> 1) & 3,
// right for eight neighbouring rows, cost 1.5 times the reads' cycles).
// A product of 8192 x 4096 x 4096 takes 139 us (2.0 POP/s; in a graph, where a
// library's bare integer product takes 129 on the same card; 143 on another;
// 151 between other kernels): the matrix units are busy 50 % of the cycles, LDS
// has no bank conflict, L2 serves 86 % of the lines, and the clock gives way
// under load (codes that are all zero: 112 us, the library's 103).  Deeper
// rings, four waves of 128 x 128 and reads further ahead of the products changed
// nothing there.
constexpr int kPartBytes = 64;

// lane l's 16 bytes at p go to LDS byte `to` + 16 * l (to: the same in all lanes).
// The compiler does not count these loads: the waits below do.  Nor can it be told
// that m0 changes (a reserved register: naming it as clobbered is warned against
// and changes no instruction); it has no use for m0 of its own in these kernels,
// which a test of their assembly holds it to.
__device__ __forceinline__ void load_to_lds(const int8_t* p, uint32_t to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(to) : "memory");
}

// waits until at most N of this wave's loads to LDS are still on their way and
// its reads of LDS are done, then for all waves
template <int N>
__device__ __forceinline__ void wait_step() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// the same where only `behind` <= B steps of LOADS loads are left
template <int B, int LOADS>
__device__ __forceinline__ void wait_last(int behind) {
  if constexpr (B > 0) {
    if (behind == B) wait_step<B * LOADS>();
    else wait_last<B - 1, LOADS>(behind);
  } else {
    wait_step<0>();
  }
}

// a wave's own loads alone: until `behind` <= B steps of LOADS loads are left
template <int B, int LOADS>
__device__ __forceinline__ void wait_own(int behind) {
  if (B == 0 || behind >= B) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(B * LOADS) : "memory");
  else wait_own<(B > 0 ? B - 1 : 0), LOADS>(behind);
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// The 16 values that a lane holds of a 32 x 32 block, rows (i & 3) + 8 * (i >>
// 2) after its first: through a buffer that begins at the block's first row
// (where rows are mapped, at the matrix's) and ends behind the last row of the
// matrix, so an access costs one 32-bit add and the hardware's range check
// leaves out the rows past the end (and rows and columns that are not there,
// whose offset is kOutside).
constexpr uint32_t kOutside = 0x80000000u;
struct BlockRows {
  __amdgpu_buffer_rsrc_t rows;
  uint32_t ld;  // bytes
  __device__ __forceinline__ BlockRows(const void* p, int size, long long ldx, int first, int end)
      : rows(__builtin_amdgcn_make_buffer_rsrc((char*)const_cast<void*>(p) + first * ldx * size, 0,
                                               (int)min(max((long long)end - first, 0ll) * ldx * size, 32 * ldx * size),
                                               0x00020000)),
        ld((uint32_t)ldx * size) {}
  // all `rows` rows of a matrix smaller than 2^31 bytes
  __device__ __forceinline__ BlockRows(const void* p, int size, long long ldx, long long count)
      : rows(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)(count * ldx * size), 0x00020000)),
        ld((uint32_t)ldx * size) {}
};
template <class F>
__device__ __forceinline__ void each_16(const uint32_t (&at)[16], F f) {
#pragma unroll
  for (int i = 0; i < 16; i++) f(i, at[i]);
}
__device__ __forceinline__ void load_16(const BlockRows& b, int type, const uint32_t (&at)[16], float (&z)[16]) {
  if (type == kFloat32)
    each_16(at, [&](int i, uint32_t o) { z[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(b.rows, o, 0, 0)); });
  else if (type == kFloat16)
    each_16(at, [&](int i, uint32_t o) { z[i] = __half2float(__ushort_as_half(__builtin_amdgcn_raw_buffer_load_b16(b.rows, o, 0, 0))); });
  else
    each_16(at, [&](int i, uint32_t o) { z[i] = __uint_as_float((uint32_t)__builtin_amdgcn_raw_buffer_load_b16(b.rows, o, 0, 0) << 16); });
}
__device__ __forceinline__ void store_16(const BlockRows& b, int type, const uint32_t (&at)[16], const float (&v)[16]) {
  if (type == kFloat32)
    each_16(at, [&](int i, uint32_t o) { __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v[i]), b.rows, o, 0, 0); });
  else if (type == kFloat16)
    each_16(at, [&](int i, uint32_t o) { __builtin_amdgcn_raw_buffer_store_b16(__half_as_ushort(__float2half(v[i])), b.rows, o, 0, 0); });
  else
    each_16(at, [&](int i, uint32_t o) { __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (__bf16)v[i]), b.rows, o, 0, 0); });
}

struct Column {  // a column's constants
  float sw, bias, gain, shift;
};
__device__ __forceinline__ Column column(const LinearInt8& a, int n) {
  Column c{a.sw[n], 0.0f, 1.0f, 0.0f};
  if (a.bias) c.bias = a.bias[n];
  if (a.gain) {
    c.gain = a.gain[n];
    c.shift = a.shift[n];
  }
  return c;
}

// Epilogue of a lane's 16 values of the block at row m0, column n of the lane
// (z: the residual's)
__device__ __forceinline__ void finish_16(const LinearInt8& a, float (&v)[16], const Column& c, const float (&z)[16]) {
#pragma unroll
  for (int i = 0; i < 16; i++) v[i] = v[i] * c.sw;
  if (a.bias) {
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = v[i] + c.bias;
  }
  if (a.relu) {
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = v[i] < 0.0f ? 0.0f : v[i];
  }
  if (a.gain) {
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = v[i] * c.gain + c.shift;
  }
  if (a.residual) {
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = a.res_scale * z[i] + v[i];
  }
}

// The same for one value
__device__ __forceinline__ void finish_one(const LinearInt8& a, float v, const Column& c, int m, int n) {
  float y = v * c.sw;
  if (a.bias) y = y + c.bias;
  if (a.relu) y = y < 0.0f ? 0.0f : y;
  if (a.gain) y = y * c.gain + c.shift;
  if (a.residual) {
    const int from = a.res_from ? a.res_from[m * a.ldres_from] : m;
    // (an absent row is not read: there may be no row at all)
    const float z = from >= 0 && from < a.res_rows ? load_float(a.residual, a.res_type, from * a.ldr + n) : 0.0f;
    y = a.res_scale * z + y;
  }
  const int to = a.out_to ? a.out_to[m * a.ldout_to] : m;
  if (to >= 0 && to < a.out_rows) store_float(a.out, a.out_type, to * a.ldo + n, y);
}

// (two waves a SIMD leave 256 registers a wave: the accumulators then stay
// where the products and the epilogue both use them, without a copy a step)
// MAPPED: rows of out or of the residual go through maps (in a kernel of its
// own: the choice at run time cost the others 5 %).
template <int TM, int TN, int WM, int WN, int ST, int KB, bool MULTI, bool MAPPED>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(2))) void linear_tile_kernel(LinearInt8 a, int tiles_m, int tiles_n) {
  constexpr int NW = WM * WN, NT = 64 * NW;
  constexpr int BM = TM / WM / 32, BN = TN / WN / 32;  // 32 x 32 blocks of a wave
  constexpr int LOADS = (TM + TN) / 16 / NW;           // load instructions of a wave for a part of K
  constexpr int PART = (TM + TN) * kPartBytes;         // LDS bytes of those
  static_assert((TM + TN) % (16 * NW) == 0, "every wave has the same number of loads");
  extern __shared__ char smem[];                       // ST x KB x [TM + TN][64], scales [taps][TM], row tables
  float* const sscale = (float*)(smem + ST * KB * PART);
  int* const srow = (int*)(sscale + a.taps * TM);
  uint32_t* const sout = (uint32_t*)(srow + (MULTI ? a.taps * TM : 0));  // mapped rows of out and residual: their bytes
  uint32_t* const sres = sout + (MAPPED && a.out_to ? TM : 0);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // workgroups b, b + 8, ... run on one XCD: each XCD gets neighbouring tiles
  // (GROUP rows of tiles, column after column), whose rows its L2 reads once
  constexpr int GROUP = 4;
  const int tiles = tiles_m * tiles_n;
  const long long block = block_id();
  if (block >= tiles) return;
  const int xcd = (int)(block & 7);
  const int t = xcd * (tiles >> 3) + min(xcd, tiles & 7) + (int)(block >> 3);
  const int g0 = t / (GROUP * tiles_n) * GROUP, gm = min(GROUP, tiles_m - g0), gt = t - g0 * tiles_n;
  const int m0 = (g0 + gt % gm) * TM, n0 = gt / gm * TN;
  // which row each output row reads; those past the count, which is not known yet, as well
  auto row_of = [&](int m, int tap) {  // -1: adds nothing
    const int row = m < a.m ? a.rows ? a.rows[m * a.ldrows + tap] : m : -1;
    return row < a.arows ? row : -1;
  };
  const int kt = a.k / kPartBytes, parts = kt * a.taps, steps = (parts + KB - 1) / KB;
  // this wave's loads: LOADS groups of 16 rows (the tile's rows of A, then of
  // W), lane l row l >> 2, chunk slot l & 3; absent rows read row 0
  const int lrow = lane >> 2, chunk = (lane & 3) ^ ((lrow >> 2) & 3);
  const int8_t* p[LOADS];
#pragma unroll
  for (int g = 0; g < LOADS; g++) {
    const int r = (wave * LOADS + g) * 16 + lrow;
    p[g] = (r < TM ? a.a + max(row_of(m0 + r, 0), 0) * a.lda : a.w + (long long)min(n0 + r - TM, a.n - 1) * a.ldw) + 16 * chunk;
  }
  if (MULTI) {  // the loads of later taps ask this table
    for (int i = tid; i < TM * a.taps; i += NT) srow[i] = row_of(m0 + i % TM, i / TM);
  }
  const int mrows = a.count ? min(a.m, *a.count) : a.m;
  if (m0 >= mrows) return;
  if (MULTI) __syncthreads();
  const uint32_t to = lds_address(smem) + wave * LOADS * 1024;
  int issued = 0, ipart = 0, ik = 0, itap = 0, ibuf = 0;
  auto issue_part = [&](int u) {  // part u of the next step
    const bool last = ik + 1 == kt;  // of the tap
#pragma unroll
    for (int g = 0; g < LOADS; g++) load_to_lds(p[g], to + (ibuf * KB + u) * PART + g * 1024);
    if (u == KB - 1) {
      issued++;
      ibuf = ibuf + 1 == ST ? 0 : ibuf + 1;
    }
    if (++ipart >= parts) return;  // (a step's parts behind the last one are loads of the last one again)
    ik = last ? 0 : ik + 1;
    itap += last;
#pragma unroll
    for (int g = 0; g < LOADS; g++) {
      const int r = (wave * LOADS + g) * 16 + lrow;
      if (MULTI && last && r < TM) p[g] = a.a + (long long)max(srow[itap * TM + r], 0) * a.lda + 16 * chunk;
      else p[g] += kPartBytes;
    }
  };
  for (int s = 0; s < ST - 1 && s < steps; s++) {
#pragma unroll
    for (int u = 0; u < KB; u++) issue_part(u);
  }
  for (int i = tid; i < TM * a.taps; i += NT) {  // read behind the first of the loop's barriers
    const int row = MULTI ? srow[i] : row_of(m0 + i, 0);
    sscale[i] = row >= 0 ? a.sa[row] : 0.0f;
  }
  const int rsize = a.res_type == kFloat32 ? 4 : 2, osize = a.out_type == kFloat32 ? 4 : 2;
  auto bytes_of = [&](const int* map, long long ld, long long rows, uint32_t row_bytes, int m) {
    const int row = m < mrows ? map[m * ld] : -1;
    return row >= 0 && row < rows ? (uint32_t)row * row_bytes : kOutside;
  };
  if (MAPPED) {
    for (int i = tid; i < TM; i += NT) {
      if (a.out_to) sout[i] = bytes_of(a.out_to, a.ldout_to, a.out_rows, (uint32_t)(a.ldo * osize), m0 + i);
      if (a.res_from) sres[i] = bytes_of(a.res_from, a.ldres_from, a.res_rows, (uint32_t)(a.ldr * rsize), m0 + i);
    }
  }

  const int r32 = lane & 31, h = lane >> 5;
  const int wm = wave / WN * (TM / WM), wn = wave % WN * (TN / WN);
  // the columns' constants, and the residual of a wave's only block, are on their way during the product
  Column col[BN];
#pragma unroll
  for (int y = 0; y < BN; y++) col[y] = column(a, min(n0 + wn + y * 32 + r32, a.n - 1));
  // where a lane's 16 values of a block lie
  auto place = [&](int x, int y, uint32_t ld, int size, const uint32_t* map, uint32_t (&at)[16]) {
    const int n = n0 + wn + y * 32 + r32;
    const uint32_t col = n < a.n ? (uint32_t)(n * size) : kOutside;
#pragma unroll
    for (int q = 0; q < 4; q++) {
      if (MAPPED && map) {
        const uint4 f = *reinterpret_cast<const uint4*>(&map[wm + x * 32 + 4 * h + 8 * q]);
        at[4 * q] = max(f.x, f.x + col);  // (a column and a row that are both outside: no wrap to inside)
        at[4 * q + 1] = max(f.y, f.y + col);
        at[4 * q + 2] = max(f.z, f.z + col);
        at[4 * q + 3] = max(f.w, f.w + col);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) at[4 * q + i] = col + (4 * h + 8 * q + i) * ld;
      }
    }
  };
  auto residual = [&](int x, int y, float (&z)[16]) {
    const BlockRows b = MAPPED && a.res_from ? BlockRows(a.residual, rsize, a.ldr, a.res_rows)
                                   : BlockRows(a.residual, rsize, a.ldr, m0 + wm + x * 32, mrows);
    uint32_t at[16];
    place(x, y, b.ld, rsize, MAPPED && a.res_from ? sres : nullptr, at);
    load_16(b, a.res_type, at, z);
  };
  float z[16];
  const bool late = BM * BN > 1 || (MAPPED && a.res_from);  // (its rows' table is read behind the loop)
  if (!late && a.residual) residual(0, 0, z);
  const int f0 = (h ^ ((r32 >> 2) & 3)) << 4, f1 = ((2 + h) ^ ((r32 >> 2) & 3)) << 4;
  intx16 acc[BM][BN];
  float v[MULTI ? BM : 1][MULTI ? BN : 1][16];
#pragma unroll
  for (int x = 0; x < BM; x++)
#pragma unroll
    for (int y = 0; y < BN; y++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        acc[x][y][i] = 0;
        if (MULTI) v[x][y][i] = 0.0f;
      }
  auto row_scales = [&](int tap, int x, float (&sc)[16]) {
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const float4 f = *reinterpret_cast<const float4*>(&sscale[tap * TM + wm + x * 32 + 4 * h + 8 * q]);
      sc[4 * q] = f.x;
      sc[4 * q + 1] = f.y;
      sc[4 * q + 2] = f.z;
      sc[4 * q + 3] = f.w;
    }
  };

  int buf = 0, k = 0, tap = 0;
  // half a part of the step in buf: what the wave reads of it, its products
  constexpr int AHEAD = BM * BN == 1 ? 4 : 1;
  intx4 fa[AHEAD][BM], fb[AHEAD][BN];
  auto fetch = [&](int i) {
    const char* const at = smem + (buf * KB + i / 2) * PART + (i & 1 ? f1 : f0);
#pragma unroll
    for (int x = 0; x < BM; x++) fa[i % AHEAD][x] = *reinterpret_cast<const intx4*>(at + (wm + r32 + x * 32) * kPartBytes);
#pragma unroll
    for (int y = 0; y < BN; y++) fb[i % AHEAD][y] = *reinterpret_cast<const intx4*>(at + (TM + wn + r32 + y * 32) * kPartBytes);
  };
  auto multiply = [&](int i, int keep) {
#pragma unroll
    for (int x = 0; x < BM; x++) fa[i % AHEAD][x] &= keep;
#pragma unroll
    for (int x = 0; x < BM; x++)
#pragma unroll
      for (int y = 0; y < BN; y++)
        acc[x][y] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[i % AHEAD][x], fb[i % AHEAD][y], acc[x][y], 0, 0, 0);
  };
  auto join = [&](int u) {  // u more parts of the tap are done: is it?
    if (!MULTI || (k += u) < kt) return;
    k = 0;
#pragma unroll
    for (int x = 0; x < BM; x++) {
      float sc[16];
      row_scales(tap, x, sc);
#pragma unroll
      for (int y = 0; y < BN; y++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          v[x][y][i] = fmaf((float)acc[x][y][i], sc[i], v[x][y][i]);
          acc[x][y][i] = 0;
        }
    }
    tap++;
  };
  for (int s = 0; s < steps; s++) {
    const int behind = issued - s - 1;  // steps in flight after this one
    if (behind >= ST - 2) wait_step<(ST - 2) * KB * LOADS>();
    else wait_last<ST - 3, KB * LOADS>(behind);
    // The next step's loads go into the buffer that every wave left before the barrier.  A wave stands still while its
    // loads are taken: with many blocks a wave they go out between its products (8192 x 4096 x 4096 147 -> 140 us), with
    // few at once, ahead of them (1999 x 777 x 1001 7.5 against 7.2).
    constexpr bool BETWEEN = BM * BN >= 8;
    const bool more = issued < steps;
    if (!BETWEEN && more) {
#pragma unroll
      for (int u = 0; u < KB; u++) issue_part(u);
    }
    if (BM * BN == 1 && KB >= (MULTI ? 4 : 2) && (!MULTI || k + KB <= kt)) {
      // A wave with one block waits for its reads of LDS: they go ahead of the products (2048 x 512 x 1024 6.3 -> 6.0
      // us, 1999 x 777 x 2 * 1001 12.4 -> 11.8).  With more blocks the products hide them (8192 x 4096 x 4096 1 %
      // slower so), and where two paths share both sets of accumulators they are copied.
#pragma unroll
      for (int i = 0; i < AHEAD - 1 && i < 2 * KB; i++) fetch(i);
#pragma unroll
      for (int i = 0; i < 2 * KB; i++) {
        if (i + AHEAD - 1 < 2 * KB) fetch(i + AHEAD - 1);
        __builtin_amdgcn_sched_barrier(0);
        multiply(i, MULTI || s * KB + i / 2 < parts ? -1 : 0);  // (a part behind the last one adds nothing)
        __builtin_amdgcn_sched_barrier(0);
      }
      join(KB);
    } else {  // part after part: a tap may end within the step
#pragma unroll
      for (int u = 0; u < KB; u++) {
        if (s * KB + u >= parts) break;
        if (BETWEEN && more) issue_part(u);
#pragma unroll
        for (int i = 2 * u; i < 2 * u + 2; i++) {
          fetch(i);
          multiply(i, -1);
        }
        join(1);
      }
    }
    buf = buf + 1 == ST ? 0 : buf + 1;
  }
#pragma unroll
  for (int x = 0; x < BM; x++) {
    float sc[16];
    if (!MULTI) row_scales(0, x, sc);
#pragma unroll
    for (int y = 0; y < BN; y++) {
      float w[16];
#pragma unroll
      for (int i = 0; i < 16; i++) w[i] = MULTI ? v[x][y][i] : fmaf((float)acc[x][y][i], sc[i], 0.0f);
      if (late && a.residual) residual(x, y, z);
      finish_16(a, w, col[y], z);
      const BlockRows b = MAPPED && a.out_to ? BlockRows(a.out, osize, a.ldo, a.out_rows)
                                   : BlockRows(a.out, osize, a.ldo, m0 + wm + x * 32, mrows);
      uint32_t at[16];
      place(x, y, b.ld, osize, MAPPED && a.out_to ? sout : nullptr, at);
      store_16(b, a.out_type, at, w);
    }
  }
}

// ---- narrow tiles
//
// Few columns a workgroup, so that the chip is full where 64 x 64 tiles are
// few: a tile of 16 * RT rows and 16 * CT columns in 16 x 16 blocks of
// v_mfma_i32_16x16x64_i8 (lane l holds row / column l & 15, bytes 16 * (l >> 4)
// of a step), whose K steps of 64 bytes the eight waves share.  No two waves
// read the same bytes, so each has a ring of ST steps in LDS of its own and
// waits for nobody until the waves' integer sums are joined, tap by tap.
// (Loaded straight into registers as the matrix instruction takes them, four
// neighbouring lanes read four rows, and a CU takes in 13 bytes a cycle instead
// of 21: 64 x 4096 x 4096 10.8 us against 7.6.)
// Rows of floats (TYPE >= 0; RT blocks cover all rows then) are quantised in
// LDS by the workgroup itself, each for itself, while its first weights are on
// their way.
constexpr int kNarrowWaves = 8, kNarrowThreads = 64 * kNarrowWaves;
constexpr int kFusedValues = 16384;  // float values (rows x taps x padded columns) that a workgroup quantises itself

template <int TYPE, int RT, int CT, int ST, int VALUES>  // TYPE < 0: codes, else up to VALUES float values
__global__ __launch_bounds__(kNarrowThreads) void linear_narrow_kernel(LinearInt8 a, QuantizeRows x, int tiles_m, int tiles_n) {
  constexpr bool FLOATS = TYPE >= 0;
  constexpr int R = 16 * RT, BLOCKS = RT * CT, LOADS = (FLOATS ? 0 : RT) + CT;
  // rings [8][ST][LOADS][16][64], sums [8][BLOCKS][256], scales [taps][R], codes: rows [taps][R]; floats: maxima
  // [taps][R] as bits, codes [m][ldl]
  extern __shared__ char smem[];
  int* const part = (int*)(smem + kNarrowWaves * ST * LOADS * 1024);
  float* const sscale = (float*)(part + kNarrowWaves * BLOCKS * 256);
  int* const srow = (int*)(sscale + a.taps * R);
  uint32_t* const smax = (uint32_t*)srow;
  char* const scode = (char*)(smax + a.taps * R);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // an XCD's tiles are neighbours, the rows of a column first: its L2 reads the weights once
  const int tiles = tiles_m * tiles_n;
  const long long block = block_id();
  if (block >= tiles) return;
  const int xcd = (int)(block & 7), t = xcd * (tiles >> 3) + min(xcd, tiles & 7) + (int)(block >> 3);
  const int m0 = t % tiles_m * R, n0 = t / tiles_m * 16 * CT;
  auto row_of = [&](int m, int tap) {  // -1: adds nothing
    const int row = m < a.m ? a.rows ? a.rows[m * a.ldrows + tap] : m : -1;
    return row < a.arows ? row : -1;
  };
  const int kt = a.k / kPartBytes, steps = kt * a.taps;
  // a load: 16 rows, lane l row l >> 2, chunk slot l & 3; absent rows read row 0
  const int lrow = lane >> 2, chunk = 16 * ((lane & 3) ^ ((lrow >> 2) & 3));
  const int8_t* wp[CT];
#pragma unroll
  for (int c = 0; c < CT; c++) wp[c] = a.w + (long long)min(n0 + 16 * c + lrow, a.n - 1) * a.ldw + chunk;
  const int8_t* p[RT];  // of the tap of the last load
  int itap = 0;
  if (!FLOATS) {
    while ((itap + 1) * kt <= wave) itap++;
#pragma unroll
    for (int b = 0; b < RT; b++)
      p[b] = a.a + max(row_of(m0 + 16 * b + lrow, min(itap, a.taps - 1)), 0) * a.lda + chunk;
  }
  const int mrows = a.count ? min(a.m, *a.count) : a.m;
  if (m0 >= mrows) return;
  if (!FLOATS && a.taps > 1) {
    for (int i = tid; i < a.taps * R; i += kNarrowThreads) srow[i] = max(row_of(m0 + i % R, i / R), 0);
    __syncthreads();
  }
  const uint32_t ring = lds_address(smem) + wave * ST * LOADS * 1024;
  int is = wave, ibuf = 0, issued = 0;
  auto issue = [&] {
    const uint32_t to = ring + ibuf * LOADS * 1024;
    if (!FLOATS) {
      if (is >= (itap + 1) * kt) {
        do itap++;
        while (is >= (itap + 1) * kt);
#pragma unroll
        for (int b = 0; b < RT; b++) p[b] = a.a + (long long)srow[itap * R + 16 * b + lrow] * a.lda + chunk;
      }
#pragma unroll
      for (int b = 0; b < RT; b++) load_to_lds(p[b] + kPartBytes * (is - itap * kt), to + (CT + b) * 1024);
    }
#pragma unroll
    for (int c = 0; c < CT; c++) load_to_lds(wp[c] + kPartBytes * is, to + c * 1024);
    ibuf = ibuf + 1 == ST ? 0 : ibuf + 1;
    is += kNarrowWaves;
    issued++;
  };
  for (int i = 0; i < ST - 1 && is < steps; i++) issue();
  // value i of a thread: t = tid + 512 * i of the blocks' 256 each, row t >> 4, column t & 15
  constexpr int EACH = (BLOCKS * 256 + kNarrowThreads - 1) / kNarrowThreads;
  auto row_in = [&](int i) { return ((tid + i * kNarrowThreads) >> 8) / CT * 16 + (tid >> 4 & 15); };
  auto col_in = [&](int i) { return ((tid + i * kNarrowThreads) >> 8) % CT * 16 + (tid & 15); };
  Column col[CT > 1 ? EACH : 1];
#pragma unroll
  for (int i = 0; i < (CT > 1 ? EACH : 1); i++) col[i] = column(a, min(n0 + col_in(i), a.n - 1));

  const int ldl = steps * kPartBytes + 16;  // 16 bytes on: rows in other banks
  if constexpr (FLOATS) {
    constexpr int N = Chunk<TYPE>::N;
    // all chunks of all rows of all taps stay in registers (LinearFloatFused)
    const int chunks = a.k / N, all = mrows * a.taps * chunks;  // past a row's end: zeros
    constexpr int HELD = VALUES / (kNarrowThreads * N);
    auto row_of_tap = [&](int q) { return a.taps == 1 ? q : q / a.taps; };  // of tap q of all rows
    Chunk<TYPE> c[HELD];
    int place[HELD];  // tap * R + row; -1: the row is absent
#pragma unroll
    for (int i = 0; i < HELD; i++) {
      const int u = tid + i * kNarrowThreads, q = u / chunks, m = row_of_tap(q), j = q - m * a.taps;
      place[i] = -1;
      if (u >= all) continue;
      const int row = row_of(m, j);
      if (row >= 0) {
        place[i] = j * R + m;
        c[i].load(x.x, row * x.ldx, (u - q * chunks) * N, x.k);
      }
    }
    for (int i = tid; i < a.taps * R; i += kNarrowThreads) smax[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < HELD; i++) {
      uint32_t top = place[i] >= 0 ? c[i].top_bits(c[i].top(0)) : 0u;
      const int one = __builtin_amdgcn_readfirstlane(place[i]);
      if (__all(place[i] == one)) {  // one atomic a wave where it holds one row
        if (one < 0) continue;
        top = wave_max(top);
        if (lane == 0) atomicMax(&smax[one], top);
      } else if (place[i] >= 0) {
        atomicMax(&smax[place[i]], top);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < HELD; i++) {
      const int u = tid + i * kNarrowThreads, q = u / chunks, m = row_of_tap(q), j = q - m * a.taps, e = (u - q * chunks) * N;
      if (u >= all) break;
      if (place[i] >= 0) {
        const RowScale r = row_scale(smax[place[i]]);
        c[i].store((int8_t*)scode + m * ldl + j * a.k + e, r);
        if (e == 0) sscale[place[i]] = r.scale;
      } else if (e == 0) {
        sscale[j * R + m] = 0.0f;  // (whatever its codes: the sum of them is finite)
      }
    }
    __syncthreads();
  } else {
    for (int i = tid; i < a.taps * R; i += kNarrowThreads) {  // read behind a join's barrier
      const int row = row_of(m0 + i % R, i / R);
      sscale[i] = row >= 0 ? a.sa[row] : 0.0f;
    }
  }

  float v[EACH];
#pragma unroll
  for (int i = 0; i < EACH; i++) v[i] = 0.0f;
  intx4 acc[RT][CT];
#pragma unroll
  for (int b = 0; b < RT; b++)
#pragma unroll
    for (int c = 0; c < CT; c++) acc[b][c] = intx4{0, 0, 0, 0};
  int tap = 0, end = kt;  // the tap's steps end there
  auto join = [&] {       // the tap's integer sums, then the row's scale
    if (tap) __syncthreads();
#pragma unroll
    for (int b = 0; b < RT; b++)
#pragma unroll
      for (int c = 0; c < CT; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          part[((wave * RT + b) * CT + c) * 256 + ((lane >> 4) * 4 + i) * 16 + (lane & 15)] = acc[b][c][i];
          acc[b][c][i] = 0;
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const int e = tid + i * kNarrowThreads;
      if (e < BLOCKS * 256) {
        int sum = 0;
#pragma unroll
        for (int u = 0; u < kNarrowWaves; u++) sum += part[u * BLOCKS * 256 + e];
        v[i] = fmaf((float)sum, sscale[tap * R + row_in(i)], v[i]);
      }
    }
    tap++;
    end += kt;
  };
  const int r16 = lane & 15;
  const char* const own = smem + wave * ST * LOADS * 1024 + r16 * kPartBytes + 16 * ((lane >> 4) ^ ((r16 >> 2) & 3));
  const char* held[RT];  // floats: a lane's row, one that is not there the last one (its sums are not used)
#pragma unroll
  for (int b = 0; b < RT; b++) held[b] = scode + min(16 * b + r16, mrows - 1) * ldl + 16 * (lane >> 4);
  int buf = 0, done = 0;
  for (int s = wave; s < steps; s += kNarrowWaves) {
    // (a wave joins a tap when it is past it: every wave joins every tap once, in order)
    while (s >= end) join();
    wait_own<ST - 2, LOADS>(issued - ++done);
    if (is < steps) issue();  // over the step before, whose reads are done
    const char* const at = own + buf * LOADS * 1024;
    intx4 fa[RT], fb[CT];
#pragma unroll
    for (int b = 0; b < RT; b++)
      fa[b] = *reinterpret_cast<const intx4*>(FLOATS ? held[b] + kPartBytes * s : at + (CT + b) * 1024);
#pragma unroll
    for (int c = 0; c < CT; c++) fb[c] = *reinterpret_cast<const intx4*>(at + c * 1024);
#pragma unroll
    for (int b = 0; b < RT; b++)
#pragma unroll
      for (int c = 0; c < CT; c++) acc[b][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[b], fb[c], acc[b][c], 0, 0, 0);
    buf = buf + 1 == ST ? 0 : buf + 1;
  }
  while (tap < a.taps) join();
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const int m = m0 + row_in(i), n = n0 + col_in(i);
    if (tid + i * kNarrowThreads < BLOCKS * 256 && m < mrows && n < a.n) finish_one(a, v[i], col[CT > 1 ? i : 0], m, n);
  }
}

// more than 64 KB of LDS has to be asked for
void AskLds(const void* kernel, size_t bytes) {
  if (bytes > 64 * 1024 &&
      hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != hipSuccess) {
    (void)hipGetLastError();
    VAMD_ERR("the device does not give a workgroup " << bytes << " bytes of LDS");
  }
}

}  // namespace

void LaunchQuantizeRows(const QuantizeRows& a, hipStream_t s) {
  if (a.m <= 0) return;
  if (a.type == kFloat32) LaunchQuantize<kFloat32>(a, s);
  else if (a.type == kFloat16) LaunchQuantize<kFloat16>(a, s);
  else LaunchQuantize<kBFloat16>(a, s);
}

void SetOffsets(FrameMap* a, const int* offsets) {
  const long long ring = (long long)a->pages * a->page;
  a->by_ring = Divider((uint32_t)ring);
  a->by_page = Divider((uint32_t)a->page);
  a->max_offset = INT_MIN;
  a->far_offsets = false;
  for (int j = 0; j < a->taps; j++) {
    a->offset[j] = offsets[j];
    a->max_offset = offsets[j] > a->max_offset ? offsets[j] : a->max_offset;
    a->far_offsets = a->far_offsets || offsets[j] > (1 << 30) || offsets[j] < -(1 << 30);
    a->offset_at[j] = (unsigned)(((long long)offsets[j] % ring + ring) % ring);
  }
}

namespace {

template <int THREADS, int EACH>
void LaunchMap(const FrameMap& a, hipStream_t s) {
  // Two rows a lane once there are enough rows for it: fewer workgroups then sum the streams (us in a graph, one / two
  // rows a lane, 4 001 streams and room for 200 050 rows of 5 entries 7.3 / 9.1, 400 100 8.5 / 9.3, 800 200 12.3 / 11.4).
  const int each = a.cap > 512 * 1024 && a.taps <= 8 ? 2 : 1;
  const long long grid = (a.cap + each * THREADS - 1) / (each * THREADS);
  if (!EACH && !grid) return;
  const unsigned lds = each * THREADS * a.taps * sizeof(int);
  auto kernel = each == 1 ? frame_map_kernel<THREADS, EACH, 1> : frame_map_kernel<THREADS, EACH, 2>;
  AskLds((const void*)kernel, lds);
  hipLaunchKernelGGL(kernel, Grid(grid ? grid : 1), dim3(THREADS), lds, s, a);
}

}  // namespace

void LaunchFrameMap(const FrameMap& a, hipStream_t s) {
  if (a.streams > kMapStreams) {
    hipLaunchKernelGGL(frame_starts_kernel, dim3(1), dim3(kStartsThreads), 0, s, a);
    LaunchMap<kMapThreads, 0>(a, s);
  } else if (a.streams > kMapThreads) {
    LaunchMap<kMapManyThreads, kMapStreams / kMapManyThreads>(a, s);
  } else {
    LaunchMap<kMapThreads, 1>(a, s);
  }
}

namespace {

template <int THREADS, int EACH>
void LaunchMaps(const FrameMaps& all, int n, long long cap, int taps, hipStream_t s) {
  const unsigned lds = THREADS * taps * sizeof(int);
  auto kernel = frame_maps_kernel<THREADS, EACH>;
  AskLds((const void*)kernel, lds);
  dim3 grid = Grid(cap ? (cap + THREADS - 1) / THREADS : 1);
  grid.z = n;
  hipLaunchKernelGGL(kernel, grid, dim3(THREADS), lds, s, all);
}

}  // namespace

void LaunchFrameMaps(const FrameMap* maps, int n, hipStream_t s) {
  for (; n > 0; maps += kMapsPerLaunch, n -= kMapsPerLaunch) {
    const int some = n < kMapsPerLaunch ? n : kMapsPerLaunch;
    FrameMaps all{};
    long long cap = 0;
    int taps = 0, streams = 0;
    for (int i = 0; i < some; i++) {
      all.map[i] = maps[i];
      cap = maps[i].cap > cap ? maps[i].cap : cap;
      taps = maps[i].taps > taps ? maps[i].taps : taps;
      streams = maps[i].streams > streams ? maps[i].streams : streams;
    }
    if (streams > kMapStreams) {
      for (int i = 0; i < some; i++) LaunchFrameMap(maps[i], s);
    } else if (streams > kMapThreads) {
      LaunchMaps<kMapManyThreads, kMapStreams / kMapManyThreads>(all, some, cap, taps, s);
    } else {
      LaunchMaps<kMapThreads, 1>(all, some, cap, taps, s);
    }
  }
}

namespace {

template <int TM, int TN, int WM, int WN, int ST, int KB, bool MULTI>
void LaunchTile(const LinearInt8& a, hipStream_t s) {
  const long long tm = ((long long)a.m + TM - 1) / TM, tn = ((long long)a.n + TN - 1) / TN;
  const size_t lds = ST * KB * (TM + TN) * kPartBytes + (size_t)TM * 4 * (a.taps * (MULTI ? 2 : 1) + (a.out_to ? 1 : 0) + (a.res_from ? 1 : 0));
  const bool mapped = a.out_to || a.res_from;
  auto kernel = mapped ? linear_tile_kernel<TM, TN, WM, WN, ST, KB, MULTI, true>
                       : linear_tile_kernel<TM, TN, WM, WN, ST, KB, MULTI, false>;
  AskLds((const void*)kernel, lds);
  hipLaunchKernelGGL(kernel, Grid(tm * tn), dim3(64 * WM * WN), lds, s, a, (int)tm, (int)tn);
}

// 64 x 64 tiles: the longer K is, the more of it a step (us in a graph, 1 / 2 /
// 4 parts): 4352 x 512 x 96 5.5 / 5.5 / 7.0, 2048 x 512 x 1024 6.8 / 6.3 / 5.9;
// four parts take 64 KB of LDS, which more than two tiles a CU miss: 4352 x 512
// x 1024 (544 tiles) 9.4 / 9.2 / 10.4.
template <bool MULTI>
void LaunchSmallTiles(const LinearInt8& a, long long tiles, hipStream_t s) {
  if (a.k * a.taps < 512) LaunchTile<64, 64, 2, 2, 3, 1, MULTI>(a, s);
  else if (tiles <= 512) LaunchTile<64, 64, 2, 2, 2, 4, MULTI>(a, s);
  else LaunchTile<64, 64, 2, 2, 3, 2, MULTI>(a, s);
}

template <int TYPE, int RT, int CT, int ST, int VALUES>
void LaunchNarrow(const LinearInt8& a, const QuantizeRows& x, hipStream_t s) {
  const long long tm = ((long long)a.m + 16 * RT - 1) / (16 * RT), tn = ((long long)a.n + 16 * CT - 1) / (16 * CT);
  const size_t lds = kNarrowWaves * (RT * CT + ST * ((TYPE < 0 ? RT : 0) + CT)) * 1024 + 16 * RT * a.taps * 8 +
                     (TYPE < 0 ? 0 : (size_t)a.m * ((size_t)a.k * a.taps + 16));
  auto kernel = linear_narrow_kernel<TYPE, RT, CT, ST, VALUES>;
  AskLds((const void*)kernel, lds);
  hipLaunchKernelGGL(kernel, Grid(tm * tn), dim3(kNarrowThreads), lds, s, a, x, (int)tm, (int)tn);
}

template <int TYPE>
void LaunchFused(const LinearInt8& a, const QuantizeRows& x, hipStream_t s) {
  // values kept in registers: 1 x 4096 x 4096 6.3 us with room for 4096 of them in the workgroup, 7.2 for 16384
  const bool more = (long long)a.m * a.taps * a.k > kFusedValues / 4;
  if (a.m <= 16 && more) LaunchNarrow<TYPE, 1, 1, 4, kFusedValues>(a, x, s);
  else if (a.m <= 16) LaunchNarrow<TYPE, 1, 1, 4, kFusedValues / 4>(a, x, s);
  else if (more) LaunchNarrow<TYPE, 2, 1, 4, kFusedValues>(a, x, s);
  else LaunchNarrow<TYPE, 2, 1, 4, kFusedValues / 4>(a, x, s);
}

}  // namespace

// Each workgroup quantises all rows: one launch up to 16384 values, chosen for
// the program that calls it from Python and waits for the calls, not the GPU (us
// a call of bf16 rows, one launch / two: 1 x 4096 x 4096 7.1 / 11.6, 4 x 4096 x
// 4096 9.1 / 11.5, 16 x 1024 x 96 8.3 / 11.7).  In a graph it gains with one or
// two rows (bf16 / fp32 rows, one launch against two: 1 x 4096 x 4096 5.6
// against 7.1 / 6.3 against 7.3, 2 x 512 x 512 4.7 against 5.9 / 4.2 against
// 5.7), costs little at 16 x 512 x 512 (6.1 against 6.2 / 7.6 against 6.0) and
// most at the end of the range (4 x 4096 x 4096 9.4 against 8.2 / 11.8 against
// 7.7, 32 x 512 x 512 8.1 against 6.3 / 10.6 against 6.0): a graph of such calls
// is better off with quantize_rows and codes.
bool LinearFloatFused(int m, int k, int taps) { return m <= 32 && (long long)m * k * taps <= kFusedValues; }

void LaunchLinearFloat(const LinearInt8& a, const QuantizeRows& x, hipStream_t s) {
  if (a.m <= 0 || a.n <= 0) return;
  if (LinearFloatFused(a.m, a.k, a.taps)) {
    if (x.type == kFloat32) LaunchFused<kFloat32>(a, x, s);
    else if (x.type == kFloat16) LaunchFused<kFloat16>(a, x, s);
    else LaunchFused<kBFloat16>(a, x, s);
    return;
  }
  LaunchQuantizeRows(x, s);
  LaunchLinearInt8(a, s);
}

void LaunchLinearInt8(const LinearInt8& a, hipStream_t s) {
  if (a.m <= 0 || a.n <= 0) return;
  // Narrow tiles as long as no CU gets two, the smallest first (us in a graph,
  // 16 x 16 / 32 x 16 / 32 x 32 / 64 x 64 tiles, m x n x k):
  //   16 x 4096 x 4096    5.1 /  5.7 / 5.8 / 10.4
  //   64 x 4096 x 4096   10.4 /  9.7 / 7.5 / 10.4
  //   128 x 512 x 512     3.6 /  3.7 / 4.2 /  4.3
  //   1088 x 96 x 1024    4.5 /  4.1 / 4.6 /  5.2
  //   1088 x 512 x 512   10.1 / 10.6 / 8.6 /  4.7
  const QuantizeRows none{};
  auto tiles = [&](int tm, int tn) { return (((long long)a.m + tm - 1) / tm) * (((long long)a.n + tn - 1) / tn); };
  if (tiles(16, 16) <= 256) return LaunchNarrow<-1, 1, 1, 3, 0>(a, none, s);
  if (tiles(32, 16) <= 256) return LaunchNarrow<-1, 2, 1, 4, 0>(a, none, s);
  if (tiles(32, 32) <= 256) return LaunchNarrow<-1, 2, 2, 3, 0>(a, none, s);
  // Else tiles as large as leaves every CU one (us in a graph, 64 x 64 / 128 x
  // 128 / 256 x 256 tiles):
  //   1999 x 777 x 1001    7.4 /  9.8 / 18.1
  //   4352 x 512 x 512     7.1 /  7.7 / 12.9
  //   2048 x 2000 x 1024  14.3 / 12.4 / 20.1
  //   13056 x 512 x 512   16.1 / 12.1 / 15.7
  //   8192 x 4096 x 1024  87.8 / 54.6 / 55.4
  //   13056 x 4096 x 1024  135 / 86.2 / 94.2
  //   4096 x 4096 x 2048  73.7 / 48.9 / 44.7
  //   16384 x 4096 x 2048  298 /  180 /  161
  //   8192 x 4096 x 4096   254 /  170 /  143
  // (K from 2048 on takes the largest; shorter ones would gain from it only with
  // very many rows, 16384 x 4096 x 1024 113 / 103, 16384 x 4096 x 512 78.7 / 73.5)
  // but short products, which the stores bound, in the smallest:
  //   4352 x 2000 x 192   11.1 / 13.8 / 13.3
  // and the largest, of which a CU holds one, only where the last round of
  // them is nearly full: 5000 x 5000 x 5000 (400 tiles) 181 / 149, but 4864 x
  // 4096 x 4096 (304) 104 / 118.
  // Several taps hold a second set of accumulators, for which the largest
  // tiles have no registers; theirs gain from 128 x 128 at short K too:
  //   13056 x 512 x 2 * 96  15.3 / 13.9
  const bool wide = tiles(128, 128) >= 256;
  const long long big = tiles(256, 256), rounds = (big + 255) / 256;
  if (a.taps > 1) {
    if (wide) LaunchTile<128, 128, 4, 2, 2, 2, true>(a, s);
    else LaunchSmallTiles<true>(a, tiles(64, 64), s);
  } else if (!wide || a.k < 256) {
    LaunchSmallTiles<false>(a, tiles(64, 64), s);
  } else if (a.k >= 2048 && 4 * big >= 3 * 256 * rounds) {
    LaunchTile<256, 256, 4, 2, 2, 2, false>(a, s);
  } else {
    LaunchTile<128, 128, 4, 2, 2, 2, false>(a, s);
  }
}

}  // namespace vamd
