// Norm over groups of channels with its activation, channels last, and its gradients:
//   n = (x - mean) / sqrt(var + eps), y = act(n weight + bias)
// mean and variance over the `width` channels of a group, of one row or of all rows of a segment.
//
// Rows by themselves: a row's group is held by 1 to 64 lanes, or by a workgroup; one read, one write.
//
// Segments: tiles of rows of one segment (attention_find.h: the host knows no length) in registers. A segment that is one tile
// is done with it. Longer ones leave their tiles' means and squares, and are read a second time, mostly from the last-level cache,
// by workgroups that merge them first (by the counts, in 64 bits: no difference of large sums). The backward pass does the
// same with the channels' sums of gz and gz n (gz: the gradient before the activation): they are the weights'
// gradients, and weighted they are the two means that gx needs.
#include "activation.h"
#include "attention_find.h"
#include "common.h"
#include "group_norm_shapes.h"
#include "x3.h"

namespace {

template <int V>
struct Vec {
  float v[V];
};

template <typename T, int V>
struct RawVec {
  typedef T Type __attribute__((ext_vector_type(V)));
};
template <typename T>
struct RawVec<T, 1> {
  typedef T Type;
};

template <typename T, int V>
__device__ __forceinline__ typename RawVec<T, V>::Type raw_load(const T* p) {
  return *reinterpret_cast<const typename RawVec<T, V>::Type*>(p);
}
template <typename T, int V>
__device__ __forceinline__ float raw_get(const typename RawVec<T, V>::Type& r, int i) {
  if constexpr (V == 1)
    return (float)r;
  else
    return (float)r[i];
}
template <typename T, int V>
__device__ __forceinline__ void raw_store(T* p, const float (&v)[V]) {
  typename RawVec<T, V>::Type r;
  if constexpr (V == 1) {
    r = (T)v[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = (T)v[i];
  }
  *reinterpret_cast<typename RawVec<T, V>::Type*>(p) = r;
}

template <typename T>
__device__ __forceinline__ float param(const void* p, int64_t i, float none) {
  return p ? (float)static_cast<const T*>(p)[i] : none;
}

// ---------------------------------------------------------------------------------------- rows by themselves

// sum over the `lanes` lanes (a power of two) that hold a row's group, or over the workgroup
template <bool WIDE>
__device__ __forceinline__ float unit_sum(float s, int lanes, float* lds) {
  if constexpr (WIDE) {
    s = wave_sum(s);
    __syncthreads();  // lds may still be read
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
  }
  for (int off = lanes >> 1; off; off >>= 1) s += __shfl_xor(s, off, 64);
  return s;
}

// A workgroup's units: lane groups q, of `at_once` groups of a row and `rows` rows.
struct GnUnits {
  int at_once, rows, q, lane;
  __device__ __forceinline__ GnUnits(const GnArgs& a) {
    const int n = kThreads / a.lanes;
    q = threadIdx.x / a.lanes;
    lane = threadIdx.x % a.lanes;
    at_once = a.groups < n ? a.groups : n;
    rows = n / at_once;
  }
};

template <typename T, int V, int NV, bool WIDE>
__global__ void __launch_bounds__(kThreads) gn_rows_kernel(GnArgs a) {
  __shared__ float lds[4];
  const GnUnits u(a);
  const int g = blockIdx.y * u.at_once + u.q % u.at_once;
  const int64_t row = (int64_t)(blockIdx.x + a.block0) * u.rows + u.q / u.at_once;
  const bool live = u.q < u.at_once * u.rows && g < a.groups && row < a.rows;
  const int64_t c0 = (int64_t)g * a.width;
  const T* x = static_cast<const T*>(a.x) + row * a.x_ld + c0;
  float v[NV][V];
  float s = 0.f;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = (u.lane + n * a.lanes) * V;
    const bool in = live && c < a.width;
    typename RawVec<T, V>::Type r{};
    if (in) r = raw_load<T, V>(x + c);
#pragma unroll
    for (int i = 0; i < V; ++i) s += v[n][i] = raw_get<T, V>(r, i);
  }
  const float mean = unit_sum<WIDE>(s, a.lanes, lds) / a.width;
  float d = 0.f;
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[n][i] -= mean;
      if ((u.lane + n * a.lanes) * V < a.width) d += v[n][i] * v[n][i];
    }
  const float inverse = 1.f / sqrtf(unit_sum<WIDE>(d, a.lanes, lds) / a.width + a.eps);
  if (!live) return;
  if (a.mean && u.lane == 0) {
    a.mean[row * a.groups + g] = mean;
    a.inverse[row * a.groups + g] = inverse;
  }
  T* y = static_cast<T*>(a.y) + row * a.channels + c0;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = (u.lane + n * a.lanes) * V;
    if (c >= a.width) break;
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
      o[i] = activation<sizeof(T) == 2>(v[n][i] * inverse * param<T>(a.weight, c0 + c + i, 1.f) + param<T>(a.bias, c0 + c + i, 0.f), a.act).value;
    raw_store<T, V>(y + c, o);
  }
}

// the same group of rows `blocks` apart; the channels' sums of gz n and gz in part [blocks, rows of a workgroup, 2, channels]
template <typename T, int V, int NV, bool WIDE>
__global__ void __launch_bounds__(kThreads) gn_rows_bwd_kernel(GnArgs a) {
  __shared__ float lds[4];
  const GnUnits u(a);
  const int g = blockIdx.y * u.at_once + u.q % u.at_once;
  const bool mine = u.q < u.at_once * u.rows && g < a.groups;
  const int64_t c0 = (int64_t)g * a.width;
  float w[NV][V], b[NV][V], gw[NV][V], gb[NV][V];
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (u.lane + n * a.lanes) * V + i;
      const bool in = mine && c < a.width;
      w[n][i] = in ? param<T>(a.weight, c0 + c, 1.f) : 0.f;
      b[n][i] = in ? param<T>(a.bias, c0 + c, 0.f) : 0.f;
      gw[n][i] = gb[n][i] = 0.f;
    }
  for (int64_t base = (int64_t)blockIdx.x * u.rows; base < a.rows; base += (int64_t)a.blocks * u.rows) {
    const int64_t row = base + u.q / u.at_once;
    const bool live = mine && row < a.rows;
    const float mean = live ? a.mean[row * a.groups + g] : 0.f, inverse = live ? a.inverse[row * a.groups + g] : 0.f;
    const T *x = static_cast<const T*>(a.x) + row * a.x_ld + c0, *gy = static_cast<const T*>(a.g) + row * a.g_ld + c0;
    float h[NV][V], z[NV][V];
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = (u.lane + n * a.lanes) * V;
      const bool in = live && c < a.width;
      typename RawVec<T, V>::Type r{}, q{};
      if (in) r = raw_load<T, V>(x + c);
      if (in) q = raw_load<T, V>(gy + c);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        h[n][i] = in ? (raw_get<T, V>(r, i) - mean) * inverse : 0.f;
        z[n][i] = in ? raw_get<T, V>(q, i) * activation<sizeof(T) == 2>(h[n][i] * w[n][i] + b[n][i], a.act).slope : 0.f;
        gw[n][i] += z[n][i] * h[n][i];
        gb[n][i] += z[n][i];
        z[n][i] *= w[n][i];
        s += z[n][i];
        t += z[n][i] * h[n][i];
      }
    }
    s = unit_sum<WIDE>(s, a.lanes, lds) / a.width;
    t = unit_sum<WIDE>(t, a.lanes, lds) / a.width;
    if (!live) continue;
    T* gx = static_cast<T*>(a.gx) + row * a.channels + c0;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = (u.lane + n * a.lanes) * V;
      if (c >= a.width) break;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = inverse * (z[n][i] - s - h[n][i] * t);
      raw_store<T, V>(gx + c, o);
    }
  }
  if (!a.part || !mine) return;
  float* p = a.part + ((int64_t)blockIdx.x * u.rows + u.q / u.at_once) * 2 * a.channels + c0;
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (u.lane + n * a.lanes) * V + i;
      if (c < a.width) {
        p[c] = gw[n][i];
        p[a.channels + c] = gb[n][i];
      }
    }
}

// Sums of the columns of part [count, 2, channels] over its rows, in a fixed order: the weights' gradients, or, in several
// blocks of rows, the rows of the next such sum.
template <typename T>
__global__ void __launch_bounds__(1024) gn_columns_kernel(const float* part, int64_t count, int64_t columns, int64_t each, float* sums,
                                                          T* gw, T* gb) {
  __shared__ float lds[32][33];
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  const int64_t c = (int64_t)blockIdx.x * 32 + tx, from = blockIdx.y * each, to = from + each < count ? from + each : count;
  float s = 0.f;
  if (c < columns) {
    int64_t r = from + ty;
    for (; r + 96 < to; r += 128) {
      const float* p = part + r * columns + c;
      s += (p[0] + p[32 * columns]) + (p[64 * columns] + p[96 * columns]);
    }
    for (; r < to; r += 32) s += part[r * columns + c];
  }
  lds[ty][tx] = s;
  __syncthreads();
  for (int n = 16; n; n >>= 1) {
    if (ty < n) lds[ty][tx] += lds[ty + n][tx];
    __syncthreads();
  }
  if (ty || c >= columns) return;
  s = lds[0][tx];
  const int64_t half = columns / 2;
  if (sums)
    sums[blockIdx.y * columns + c] = s;
  else if (c < half)
    gw[c] = (T)s;
  else
    gb[c - half] = (T)s;
}

// ---------------------------------------------------------------------------------------- segments

// A workgroup's share of the channels [c0, c0 + nc), `tx` vectors of a row (NV apart from each other by the workgroup's width),
// and a thread's place in it.
template <int V, int NV>
struct GnPlace {
  int c0, nc, groups, x, y, step;
  float per;  // groups per channel
  bool in;
  __device__ __forceinline__ GnPlace(const GnArgs& a) {
    c0 = blockIdx.y * a.chunk;
    nc = min(a.chunk, a.channels - c0);
    groups = nc / a.width;
    per = 1.f / a.width;
    step = NV > 1 ? 1 : kThreads / a.tx;
    x = NV > 1 ? threadIdx.x : threadIdx.x % a.tx;
    y = NV > 1 ? 0 : threadIdx.x / a.tx;
    in = y < step;
  }
  __device__ __forceinline__ int column(int n) const { return (x + n * kThreads) * V; }  // within the share
  __device__ __forceinline__ bool has(int n) const { return in && column(n) < nc; }
  // channel / width, for fewer than 2^13 channels: the half keeps the rounded product off the whole numbers
  __device__ __forceinline__ int group(int channel) const { return (int)(((float)channel + 0.5f) * per); }
};

// Sums over the share's groups of `count` rows of values per channel in lds [count, nc]: out[g], in the same order for every call.
// Power of two lanes a group.
__device__ __forceinline__ void group_sums(const float* lds, int count, int nc, int width, int groups, float* out) {
  int lanes = 64;
  while (lanes > 1 && lanes * groups > kThreads) lanes >>= 1;
  const int lane = threadIdx.x % lanes, total = count * width, each = kThreads / lanes;
  const float per = 1.f / width;
  for (int g = threadIdx.x / lanes; g < max(groups, each); g += each) {  // several lanes a group: one pass, all take part
    float s = 0.f;
    if (g < groups)
      for (int i = lane; i < total; i += lanes) {
        const int r = (int)(((float)i + 0.5f) * per);  // i / width (fewer than 2^14 values)
        s += lds[r * nc + g * width + (i - r * width)];
      }
    for (int off = lanes >> 1; off; off >>= 1) s += __shfl_xor(s, off, 64);
    if (lane == 0 && g < groups) out[g] = s;
  }
}

struct GnTile {
  int segment;         // extended: 0 and segments + 1 are the rows outside
  int64_t start, rows, first;
  bool real, whole;
};

__device__ __forceinline__ GnTile gn_tile(const GnArgs& a, int64_t number) {
  GnTile t;
  t.segment = attn_find(a.off, a.segments, a.rows, 1, a.tile_rows, number, &t.first, WaveLanes());
  t.start = attn_start(a.off, a.segments, a.rows, t.segment);
  t.rows = attn_start(a.off, a.segments, a.rows, t.segment + 1) - t.start;
  t.real = t.segment >= 1 && t.segment <= a.segments;
  t.whole = t.rows <= a.tile_rows;
  return t;
}

// Tiles of long segments, for the second read, where there are few beside the tiles: those of the first read, the last one first, each on
// the XCD that read it (workgroup w runs on XCD w % 8), whose L2 holds what was read last (65 536 rows of 320, bf16: 38 -> 35 us).
__device__ __forceinline__ GnTile gn_long_tile(const GnArgs& a, int64_t number);

__device__ __forceinline__ GnTile gn_second_tile(const GnArgs& a, int64_t number) {
  if (!a.again) return gn_long_tile(a, number);
  const int64_t b = number & 7, group = number >> 3;
  return gn_tile(a, ((a.again >> 3) - 1 - group) * 8 + b);
}

// Where there are many: numbers from floor(2 start / tile) on, of which such a segment owns at least as many as it has tiles, and
// a shorter one any.
__device__ __forceinline__ GnTile gn_long_tile(const GnArgs& a, int64_t number) {
  GnTile t;
  const auto num = [&](int i) { return 2 * attn_start(a.off, a.segments, a.rows, i) / a.tile_rows; };
  t.segment = attn_last(a.segments + 2, number, num, WaveLanes());
  t.start = attn_start(a.off, a.segments, a.rows, t.segment);
  t.rows = attn_start(a.off, a.segments, a.rows, t.segment + 1) - t.start;
  t.real = t.segment >= 1 && t.segment <= a.segments;
  t.whole = t.rows <= a.tile_rows;
  const int64_t tile = number - num(t.segment);
  t.first = tile < 0 ? INT64_MAX : tile * a.tile_rows;
  return t;
}

template <typename T, int V, int NV, int NR>
struct GnRegs {
  typename RawVec<T, V>::Type r[NR][NV];
  // rows and columns past the end: the last row, or the first column, again
  __device__ __forceinline__ void load(const GnPlace<V, NV>& p, const T* x, int64_t ld, int rows) {
#pragma unroll
    for (int k = 0; k < NR; ++k)
#pragma unroll
      for (int n = 0; n < NV; ++n)
        r[k][n] = raw_load<T, V>(x + min(p.y + k * p.step, rows - 1) * ld + p.c0 + (p.has(n) ? p.column(n) : 0));
  }
  __device__ __forceinline__ float get(int k, int n, int i) const { return raw_get<T, V>(r[k][n], i); }
};

// per channel of this thread: the group's value from lds
template <int V, int NV>
__device__ __forceinline__ void spread(const GnPlace<V, NV>& p, const float* of_group, float (&v)[NV][V]) {
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) v[n][i] = of_group[p.has(n) ? p.group(p.column(n) + i) : 0];
}

// A parameter's channels of this thread; `wide`: in vectors, which its address and the other's allow.
template <typename T, int V, int NV>
__device__ __forceinline__ void spread_param(const GnPlace<V, NV>& p, const void* src, int wide, float none, float (&v)[NV][V]) {
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int at = p.c0 + (p.has(n) ? p.column(n) : 0);
    typename RawVec<T, V>::Type r{};
    if (src && wide) r = raw_load<T, V>(static_cast<const T*>(src) + at);
#pragma unroll
    for (int i = 0; i < V; ++i) v[n][i] = src && wide ? raw_get<T, V>(r, i) : param<T>(src, at + i, none);
  }
}

// values per channel, a row of lds for each of the workgroup's rows of threads
template <int V, int NV>
__device__ __forceinline__ void put_channels(const GnPlace<V, NV>& p, float* lds, const float (&v)[NV][V]) {
#pragma unroll
  for (int n = 0; n < NV; ++n)
    if (p.has(n))
#pragma unroll
      for (int i = 0; i < V; ++i) lds[p.y * p.nc + p.column(n) + i] = v[n][i];
}

template <typename T, int V, int NV, int NR>
__device__ __forceinline__ void write_zero(const GnPlace<V, NV>& p, T* y, int64_t ld, int rows) {
  const float zero[V] = {};
#pragma unroll
  for (int k = 0; k < NR; ++k)
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int row = p.y + k * p.step;
      if (p.has(n) && row < rows) raw_store<T, V>(y + row * ld + p.c0 + p.column(n), zero);
    }
}

template <typename T, int V, int NV, int NR>
__device__ __forceinline__ void write_norm(const GnArgs& a, const GnPlace<V, NV>& p, const GnRegs<T, V, NV, NR>& x, T* y, int rows,
                                           const float (&mean)[NV][V], const float (&inverse)[NV][V]) {
  float w[NV][V], b[NV][V];
  spread_param<T, V, NV>(p, a.weight, a.params_wide, 1.f, w);
  spread_param<T, V, NV>(p, a.bias, a.params_wide, 0.f, b);
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) w[n][i] *= inverse[n][i];
#pragma unroll
  for (int k = 0; k < NR; ++k)
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int row = p.y + k * p.step;
      if (!p.has(n) || row >= rows) continue;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = activation<sizeof(T) == 2>((x.get(k, n, i) - mean[n][i]) * w[n][i] + b[n][i], a.act).value;
      raw_store<T, V>(y + (int64_t)row * a.channels + p.c0 + p.column(n), o);
    }
}

// First read. part: [tiles, groups, 2], mean and sum of squared distances of a tile of a longer segment.
template <typename T, int V, int NV, int NR>
__global__ void __launch_bounds__(kThreads) gn_tile_kernel(GnArgs a) {
  extern __shared__ float lds[];  // [rows of threads, share], then the groups' values twice
  const GnPlace<V, NV> p(a);
  const int64_t number = (int64_t)blockIdx.x + a.block0;
  const GnTile t = gn_tile(a, number);
  if (t.first >= t.rows) return;
  const int rows = (int)(t.rows - t.first < a.tile_rows ? t.rows - t.first : a.tile_rows);
  const int64_t row0 = t.start + t.first;
  T* y = static_cast<T*>(a.y) + row0 * a.channels;
  if (!t.real) return write_zero<T, V, NV, NR>(p, y, a.channels, rows);
  GnRegs<T, V, NV, NR> x;
  x.load(p, static_cast<const T*>(a.x) + row0 * a.x_ld, a.x_ld, rows);
  float* of_group = lds + p.step * p.nc;
  const float count = (float)((int64_t)rows * a.width);
  float s[NV][V];
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s[n][i] = 0.f;
#pragma unroll
      for (int k = 0; k < NR; ++k) s[n][i] += p.y + k * p.step < rows ? x.get(k, n, i) : 0.f;
    }
  put_channels<V, NV>(p, lds, s);
  __syncthreads();
  group_sums(lds, p.step, p.nc, a.width, p.groups, of_group);
  __syncthreads();
  float mean[NV][V];
  spread<V, NV>(p, of_group, mean);
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      mean[n][i] /= count;
      s[n][i] = 0.f;
#pragma unroll
      for (int k = 0; k < NR; ++k) {
        const float d = p.y + k * p.step < rows ? x.get(k, n, i) - mean[n][i] : 0.f;
        s[n][i] += d * d;
      }
    }
  put_channels<V, NV>(p, lds, s);
  __syncthreads();
  float* squares = of_group + p.groups;
  group_sums(lds, p.step, p.nc, a.width, p.groups, squares);
  __syncthreads();
  const int g0 = p.c0 / a.width;
  if (!t.whole) {
    for (int g = threadIdx.x; g < p.groups; g += kThreads) {
      float2* out = reinterpret_cast<float2*>(a.part) + number * a.groups + g0 + g;
      *out = make_float2(of_group[g] / count, squares[g]);
    }
    return;
  }
  float inverse[NV][V];
  spread<V, NV>(p, squares, inverse);
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) inverse[n][i] = 1.f / sqrtf(inverse[n][i] / count + a.eps);
  if (a.mean)
    for (int g = threadIdx.x; g < p.groups; g += kThreads) {
      const int64_t at = (int64_t)(t.segment - 1) * a.groups + g0 + g;
      a.mean[at] = of_group[g] / count;
      a.inverse[at] = 1.f / sqrtf(squares[g] / count + a.eps);
    }
  write_norm<T, V, NV, NR>(a, p, x, y, rows, mean, inverse);
}

__device__ __forceinline__ bool merged_apart(const GnArgs& a, int64_t rows) { return a.merge && rows > (int64_t)kMergeTiles * a.tile_rows; }

struct GnStats {
  float x, y;
};

// Of group g of a longer segment, by `lanes` (a power of two) lanes that all call it: mean and inverse, or the two means of the
// backward pass. `tile`: number of its first tile.
template <bool BACK>
__device__ __forceinline__ GnStats merge(const GnArgs& a, int64_t tile, int64_t rows, int g, int lane, int lanes) {
  const int64_t tiles = (rows + a.tile_rows - 1) / a.tile_rows;
  const float2* part = reinterpret_cast<const float2*>(a.part) + tile * a.groups + g;
  const double total = (double)rows * a.width;
  double s = 0.0, q = 0.0;
  if (BACK) {
    for (int64_t k = lane; k < tiles; k += lanes) {
      const float2 v = part[k * a.groups];
      s += v.x;
      q += v.y;
    }
  } else {
    const double full = (double)a.tile_rows * a.width, last = (double)(rows - (tiles - 1) * a.tile_rows) * a.width;
    const float pivot = part[0].x;
    for (int64_t k = lane; k < tiles; k += lanes) {
      const float2 v = part[k * a.groups];
      const double d = (double)v.x - pivot, n = k == tiles - 1 ? last : full;
      s += d * n;
      q += v.y + d * d * n;
    }
  }
  for (int off = lanes >> 1; off; off >>= 1) {
    s += __shfl_xor(s, off, 64);
    q += __shfl_xor(q, off, 64);
  }
  if (BACK) return {(float)(s / total), (float)(q / total)};
  const double mean = s / total, square = q / total - mean * mean;
  return {(float)(part[0].x + mean), (float)(1.0 / sqrt((square > 0.0 || square != square ? square : 0.0) + (double)a.eps))};
}

// The segments of many tiles, a wave a group. A workgroup a segment, or, where there are more segments than could have so many tiles,
// numbers from floor(start / (kMergeTiles tiles)) on, of which such a segment owns one at least.
template <bool BACK>
__global__ void __launch_bounds__(kThreads) gn_merge_kernel(GnArgs a, float* x, float* y, int stride, int by_number) {
  const int64_t number = (int64_t)blockIdx.x + a.block0;
  int i = (int)number + 1;
  const auto num = [&](int i) { return attn_start(a.off, a.segments, a.rows, i) / ((int64_t)kMergeTiles * a.tile_rows); };
  if (by_number) i = attn_last(a.segments + 2, number, num, WaveLanes());
  const int64_t start = attn_start(a.off, a.segments, a.rows, i), rows = attn_start(a.off, a.segments, a.rows, i + 1) - start;
  if (i < 1 || i > a.segments || !merged_apart(a, rows) || (by_number && num(i) != number)) return;
  const int g = blockIdx.y * 4 + threadIdx.x / 64, lane = threadIdx.x & 63;
  if (g >= a.groups) return;
  const GnStats s = merge<BACK>(a, start / a.tile_rows + i, rows, g, lane, 64);
  if (lane) return;
  x[((int64_t)(i - 1) * a.groups + g) * stride] = s.x;
  y[((int64_t)(i - 1) * a.groups + g) * stride] = s.y;
}

// the same for the share's groups, into lds [2, groups], by the workgroup
template <bool BACK>
__device__ __forceinline__ void merge_share(const GnArgs& a, const GnTile& t, int g0, int groups, float* lds) {
  int lanes = 64;
  while (lanes > 1 && lanes * groups > kThreads) lanes >>= 1;
  const int lane = threadIdx.x % lanes, each = kThreads / lanes;
  for (int g = threadIdx.x / lanes; g < max(groups, each); g += each) {  // several lanes a group: one pass, all take part
    const GnStats s = merge<BACK>(a, t.start / a.tile_rows + t.segment, t.rows, g0 + min(g, groups - 1), lane, lanes);
    if (lane == 0 && g < groups) {
      lds[g] = s.x;
      lds[groups + g] = s.y;
    }
  }
  __syncthreads();
}

// the share's groups' values of a segment from memory [segments, groups] (or interleaved, stride 2) into lds [2, groups]
__device__ __forceinline__ void load_share(const float* x, const float* y, int stride, int64_t at, int groups, float* lds) {
  for (int g = threadIdx.x; g < groups; g += kThreads) {
    lds[g] = x[(at + g) * stride];
    lds[groups + g] = y[(at + g) * stride];
  }
  __syncthreads();
}

// Second read of the longer segments.
template <typename T, int V, int NV, int NR>
__global__ void __launch_bounds__(kThreads) gn_apply_kernel(GnArgs a) {
  extern __shared__ float lds[];  // [2, groups of the share]
  const GnPlace<V, NV> p(a);
  const GnTile t = gn_second_tile(a, (int64_t)blockIdx.x + a.block0);
  if (!t.real || t.whole || t.first >= t.rows) return;
  const int rows = (int)(t.rows - t.first < a.tile_rows ? t.rows - t.first : a.tile_rows);
  const int64_t row0 = t.start + t.first;
  GnRegs<T, V, NV, NR> x;
  x.load(p, static_cast<const T*>(a.x) + row0 * a.x_ld, a.x_ld, rows);
  float mean[NV][V], inverse[NV][V];
  const int g0 = p.c0 / a.width;
  if (merged_apart(a, t.rows)) {
    load_share(a.mean, a.inverse, 1, (int64_t)(t.segment - 1) * a.groups + g0, p.groups, lds);
  } else {
    merge_share<false>(a, t, g0, p.groups, lds);
    if (t.first == 0)
      for (int g = threadIdx.x; g < p.groups; g += kThreads) {
        a.mean[(int64_t)(t.segment - 1) * a.groups + g0 + g] = lds[g];
        a.inverse[(int64_t)(t.segment - 1) * a.groups + g0 + g] = lds[p.groups + g];
      }
  }
  spread<V, NV>(p, lds, mean);
  spread<V, NV>(p, lds + p.groups, inverse);
  write_norm<T, V, NV, NR>(a, p, x, static_cast<T*>(a.y) + row0 * a.channels, rows, mean, inverse);
}

// gx of a tile, some rows at a time: the two means over its segment's group in s (of gz w) and q (of gz w n)
template <typename T, int V, int NV, int NR>
__device__ __forceinline__ void write_grad(const GnArgs& a, const GnPlace<V, NV>& p, int64_t row0, int rows, const float (&mean)[NV][V],
                                           const float (&inverse)[NV][V], const float (&w)[NV][V], const float (&b)[NV][V],
                                           const float (&s)[NV][V], const float (&q)[NV][V]) {
  for (int r0 = 0; r0 < rows; r0 += a.part_rows) {
    GnRegs<T, V, NV, NR> x, gy;
    x.load(p, static_cast<const T*>(a.x) + (row0 + r0) * a.x_ld, a.x_ld, rows - r0);
    gy.load(p, static_cast<const T*>(a.g) + (row0 + r0) * a.g_ld, a.g_ld, rows - r0);
    T* gx = static_cast<T*>(a.gx) + (row0 + r0) * a.channels;
#pragma unroll
    for (int k = 0; k < NR; ++k)
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int row = p.y + k * p.step;
        if (!p.has(n) || row >= rows - r0) continue;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float h = (x.get(k, n, i) - mean[n][i]) * inverse[n][i];
          const float z = gy.get(k, n, i) * activation<sizeof(T) == 2>(h * w[n][i] + b[n][i], a.act).slope * w[n][i];
          o[i] = inverse[n][i] * (z - s[n][i] - h * q[n][i]);
        }
        raw_store<T, V>(gx + (int64_t)row * a.channels + p.c0 + p.column(n), o);
        __builtin_amdgcn_sched_barrier(0);
      }
  }
}

template <typename T, int V, int NV, int NR>
__device__ __forceinline__ void write_zeros(const GnArgs& a, const GnPlace<V, NV>& p, T* to, int rows) {
  for (int r0 = 0; r0 < rows; r0 += a.part_rows)
    write_zero<T, V, NV, NR>(p, to + (int64_t)r0 * a.channels, a.channels, min(a.part_rows, rows - r0));
}

// First read of the backward pass. columns: [tiles, 2, channels], the channels' sums of gz n and gz; part: [tiles, groups, 2], the
// groups' of gz w and gz w n.
template <typename T, int V, int NV, int NR>
__global__ void __launch_bounds__(kThreads) gn_tile_bwd_kernel(GnArgs a, float* columns) {
  extern __shared__ float lds[];  // [2, rows of threads, share], then the groups' values twice
  const GnPlace<V, NV> p(a);
  const int64_t number = (int64_t)blockIdx.x + a.block0;
  const GnTile t = gn_tile(a, number);
  columns += number * 2 * a.channels + p.c0;
  if (t.first >= t.rows || !t.real) {
    for (int c = threadIdx.x; c < p.nc; c += kThreads) columns[c] = columns[a.channels + c] = 0.f;
    if (t.first >= t.rows) return;
  }
  const int rows = (int)(t.rows - t.first < a.tile_rows ? t.rows - t.first : a.tile_rows);
  const int64_t row0 = t.start + t.first;
  if (!t.real) return write_zeros<T, V, NV, NR>(a, p, static_cast<T*>(a.gx) + row0 * a.channels, rows);
  float mean[NV][V], inverse[NV][V], w[NV][V], b[NV][V], gw[NV][V], gb[NV][V];
  float* of_group = lds + 2 * p.step * p.nc;
  load_share(a.mean, a.inverse, 1, (int64_t)(t.segment - 1) * a.groups + p.c0 / a.width, p.groups, of_group);
  spread<V, NV>(p, of_group, mean);
  spread<V, NV>(p, of_group + p.groups, inverse);
  spread_param<T, V, NV>(p, a.weight, a.params_wide, 1.f, w);
  spread_param<T, V, NV>(p, a.bias, a.params_wide, 0.f, b);
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) gw[n][i] = gb[n][i] = 0.f;
  for (int r0 = 0; r0 < rows; r0 += a.part_rows) {
    GnRegs<T, V, NV, NR> x, gy;
    x.load(p, static_cast<const T*>(a.x) + (row0 + r0) * a.x_ld, a.x_ld, rows - r0);
    gy.load(p, static_cast<const T*>(a.g) + (row0 + r0) * a.g_ld, a.g_ld, rows - r0);
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      const bool in = p.y + k * p.step < rows - r0;
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float h = (x.get(k, n, i) - mean[n][i]) * inverse[n][i];
          const float z = (in ? gy.get(k, n, i) : 0.f) * activation<sizeof(T) == 2>(h * w[n][i] + b[n][i], a.act).slope;
          gw[n][i] += z * h;
          gb[n][i] += z;
        }
      __builtin_amdgcn_sched_barrier(0);  // a row after the other: all at once took 256 registers
    }
  }
  const int plane = p.step * p.nc;
  put_channels<V, NV>(p, lds, gw);
  put_channels<V, NV>(p, lds + plane, gb);
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.nc; i += kThreads) {
    const int which = i >= p.nc, c = i - which * p.nc;
    float* of = lds + which * plane + c;
    float s = 0.f;
    for (int y = 0; y < p.step; ++y) s += of[y * p.nc];
    columns[which * a.channels + c] = s;
    *of = s * param<T>(a.weight, p.c0 + c, 1.f);  // the channel's first row has been read
  }
  __syncthreads();
  group_sums(lds, 1, p.nc, a.width, p.groups, of_group);
  group_sums(lds + plane, 1, p.nc, a.width, p.groups, of_group + p.groups);
  __syncthreads();
  if (!t.whole) {
    for (int g = threadIdx.x; g < p.groups; g += kThreads)
      reinterpret_cast<float2*>(a.part)[number * a.groups + p.c0 / a.width + g] = make_float2(of_group[p.groups + g], of_group[g]);
    return;
  }
  const float count = (float)((int64_t)rows * a.width);
  float s[NV][V], q[NV][V];
  spread<V, NV>(p, of_group + p.groups, s);
  spread<V, NV>(p, of_group, q);
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s[n][i] /= count;
      q[n][i] /= count;
    }
  write_grad<T, V, NV, NR>(a, p, row0, rows, mean, inverse, w, b, s, q);
}

template <typename T, int V, int NV, int NR>
__global__ void __launch_bounds__(kThreads) gn_apply_bwd_kernel(GnArgs a, const float* means) {
  extern __shared__ float lds[];  // [4, groups of the share]
  const GnPlace<V, NV> p(a);
  const GnTile t = gn_second_tile(a, (int64_t)blockIdx.x + a.block0);
  if (!t.real || t.whole || t.first >= t.rows) return;
  const int rows = (int)(t.rows - t.first < a.tile_rows ? t.rows - t.first : a.tile_rows);
  const int64_t row0 = t.start + t.first;
  float mean[NV][V], inverse[NV][V], w[NV][V], b[NV][V], s[NV][V], q[NV][V];
  const int g0 = p.c0 / a.width;
  const int64_t at = (int64_t)(t.segment - 1) * a.groups + g0;
  load_share(a.mean, a.inverse, 1, at, p.groups, lds + 2 * p.groups);
  if (merged_apart(a, t.rows))
    load_share(means, means + 1, 2, at, p.groups, lds);
  else
    merge_share<true>(a, t, g0, p.groups, lds);
  spread<V, NV>(p, lds, s);
  spread<V, NV>(p, lds + p.groups, q);
  spread<V, NV>(p, lds + 2 * p.groups, mean);
  spread<V, NV>(p, lds + 3 * p.groups, inverse);
  spread_param<T, V, NV>(p, a.weight, a.params_wide, 1.f, w);
  spread_param<T, V, NV>(p, a.bias, a.params_wide, 0.f, b);
  write_grad<T, V, NV, NR>(a, p, row0, rows, mean, inverse, w, b, s, q);
}

// ---------------------------------------------------------------------------------------- host

constexpr int64_t kMostBlocks = 1 << 22;

// more workgroups than one launch takes go in several, each told its first one
template <typename Launch>
int in_launches(GnArgs& a, int64_t blocks, const Launch& launch) {
  for (int64_t first = 0; first < blocks; first += kMostBlocks) {
    a.block0 = (uint32_t)first;
    launch((unsigned)(blocks - first < kMostBlocks ? blocks - first : kMostBlocks));
    FMD_CHECK_LAUNCH();
  }
  return FMD_OK;
}

// fn(vector, vectors of a lane, wide) as constants
template <typename T, typename Fn>
int with_rows(const RowShape& s, const Fn& fn) {
#define GN_ROWS(V, NV, WIDE) return fn(std::integral_constant<int, V>{}, std::integral_constant<int, NV>{}, std::integral_constant<bool, WIDE>{})
#define GN_ROWS_V(V, MOST)                                                    \
  if (s.v == V) {                                                             \
    if (!s.wide && s.nv == 1) GN_ROWS(V, 1, false);                           \
    if (!s.wide && s.nv == 2) GN_ROWS(V, 2, false);                           \
    if (!s.wide && s.nv <= 4) GN_ROWS(V, 4, false);                           \
    if (s.nv <= MOST) GN_ROWS(V, MOST, true);                                 \
  }
  if constexpr (sizeof(T) == 2) { GN_ROWS_V(8, 4) }
  GN_ROWS_V(4, 8)
  GN_ROWS_V(2, 16)
  GN_ROWS_V(1, 32)
#undef GN_ROWS_V
#undef GN_ROWS
  return FMD_EUNSUPPORTED;
}

template <typename T, typename Fn>
int with_tiles(const TileShape& s, const Fn& fn) {
#define GN_TILE(V, NV, NR) return fn(std::integral_constant<int, V>{}, std::integral_constant<int, NV>{}, std::integral_constant<int, NR>{})
#define GN_TILES(V, NR)                                \
  if (s.v == V && s.nv == 1) {                         \
    if (s.nr == NR) GN_TILE(V, 1, NR);                 \
    if (s.nr == NR / 2) GN_TILE(V, 1, NR / 2);         \
    if (s.nr == NR / 4) GN_TILE(V, 1, NR / 4);         \
  }                                                    \
  if (s.v == V && s.nv == 4) GN_TILE(V, 4, (V < 4 ? 8 / V : 2)); \
  if (s.v == V && s.nv == 32 / V) GN_TILE(V, 32 / V, 2)
  if constexpr (sizeof(T) == 2) { GN_TILES(8, 8); }
  GN_TILES(4, 16);
  GN_TILES(2, 32);
  GN_TILES(1, 32);
#undef GN_TILES
#undef GN_TILE
  return FMD_EUNSUPPORTED;
}

template <typename T>
int norm(GnArgs a, hipStream_t stream) {
  if (!a.off) {
    const RowShape s = row_shape(a, sizeof(T));
    a.lanes = s.lanes;
    const int at_once = row_groups(a, s), rows = kThreads / s.lanes / at_once;
    const unsigned y = (unsigned)fmd_cdiv(a.groups, at_once);
    FMD_REQUIRE(y < 65536);
    return with_rows<T>(s, [&](auto v, auto nv, auto wide) {
      return in_launches(a, fmd_cdiv(a.rows, rows), [&](unsigned blocks) {
        gn_rows_kernel<T, decltype(v)::value, decltype(nv)::value, decltype(wide)::value><<<dim3(blocks, y), kThreads, 0, stream>>>(a);
      });
    });
  }
  const TileShape s = tile_shape(a, sizeof(T), false);
  FMD_REQUIRE(s.chunks < 65536);
  set_tiles(a, s, sizeof(T));
  return with_tiles<T>(s, [&](auto v, auto nv, auto nr) {
    constexpr int V = decltype(v)::value, NV = decltype(nv)::value, NR = decltype(nr)::value;
    int status = in_launches(a, tile_count(a, s), [&](unsigned blocks) {
      gn_tile_kernel<T, V, NV, NR><<<dim3(blocks, s.chunks), kThreads, s.lds, stream>>>(a);
    });
    if (status || a.rows <= s.rows) return status;  // no segment is longer than a tile
    if (a.merge) {
      const int64_t numbers = a.rows / (kMergeTiles * s.rows);
      const int by_number = numbers < a.segments;
      status = in_launches(a, by_number ? numbers : a.segments, [&](unsigned blocks) {
        gn_merge_kernel<false><<<dim3(blocks, (a.groups + 3) / 4), kThreads, 0, stream>>>(a, a.mean, a.inverse, 1, by_number);
      });
      if (status) return status;
    }
    return in_launches(a, second_count(a, s), [&](unsigned blocks) {
      gn_apply_kernel<T, V, NV, NR><<<dim3(blocks, s.chunks), kThreads, 2 * (s.chunk / a.width) * 4, stream>>>(a);
    });
  });
}

// rows of the weights' last sum; from kColumnRows on, blocks of them are summed first
constexpr int64_t kColumnRows = 1024, kColumnBlocks = 64;

template <typename T>
int columns(const float* part, int64_t count, int64_t channels, float* sums, void* gw, void* gb, hipStream_t stream) {
  const unsigned x = (unsigned)fmd_cdiv(2 * channels, 32);
  if (count > kColumnRows) {
    const int64_t each = fmd_cdiv(count, kColumnBlocks), blocks = fmd_cdiv(count, each);
    gn_columns_kernel<T><<<dim3(x, (unsigned)blocks), 1024, 0, stream>>>(part, count, 2 * channels, each, sums, nullptr, nullptr);
    FMD_CHECK_LAUNCH();
    part = sums;
    count = blocks;
  }
  gn_columns_kernel<T><<<dim3(x, 1), 1024, 0, stream>>>(part, count, 2 * channels, count, nullptr, static_cast<T*>(gw),
                                                        static_cast<T*>(gb));
  FMD_CHECK_LAUNCH();
  return FMD_OK;
}

// floats of the backward pass's scratch: the channels' sums, the groups' of tiles, the longest segments' means, the sums of blocks
struct BackSpace {
  int64_t columns, part, means, sums;
};

BackSpace back_space(const GnArgs& a, int size) {
  BackSpace s{};
  if (!a.off) {
    const RowShape r = row_shape(a, size);
    s.columns = row_blocks(a, r) * (kThreads / r.lanes / row_groups(a, r)) * 2 * a.channels;
  } else {
    const int64_t tiles = tile_count(a, tile_shape(a, size, true));
    s.columns = tiles * 2 * a.channels;
    s.part = tiles * 2 * a.groups;
    s.means = 2 * (int64_t)a.segments * a.groups;
  }
  s.sums = kColumnBlocks * 2 * a.channels;
  return s;
}

template <typename T>
int norm_bwd(GnArgs a, float* work, void* gw, void* gb, hipStream_t stream) {
  const BackSpace space = back_space(a, sizeof(T));
  float *part = work, *means = work + space.columns + space.part, *sums = means + space.means;
  a.part = a.off ? work + space.columns : part;
  if (!a.off) {
    const RowShape s = row_shape(a, sizeof(T));
    a.lanes = s.lanes;
    const int at_once = row_groups(a, s), rows = kThreads / s.lanes / at_once;
    const unsigned y = (unsigned)fmd_cdiv(a.groups, at_once);
    FMD_REQUIRE(y < 65536);
    a.blocks = (int32_t)row_blocks(a, s);
    if (!gw) a.part = nullptr;
    const int status = with_rows<T>(s, [&](auto v, auto nv, auto wide) {
      gn_rows_bwd_kernel<T, decltype(v)::value, decltype(nv)::value, decltype(wide)::value><<<dim3(a.blocks, y), kThreads, 0, stream>>>(a);
      FMD_CHECK_LAUNCH();
      return (int)FMD_OK;
    });
    if (status || !gw) return status;
    return columns<T>(part, (int64_t)a.blocks * rows, a.channels, sums, gw, gb, stream);
  }
  const TileShape s = tile_shape(a, sizeof(T), true);
  FMD_REQUIRE(s.chunks < 65536);
  set_tiles(a, s, sizeof(T));
  const int status = with_tiles<T>(s, [&](auto v, auto nv, auto nr) {
    constexpr int V = decltype(v)::value, NV = decltype(nv)::value, NR = decltype(nr)::value;
    int status = in_launches(a, tile_count(a, s), [&](unsigned blocks) {
      gn_tile_bwd_kernel<T, V, NV, NR><<<dim3(blocks, s.chunks), kThreads, s.lds, stream>>>(a, part);
    });
    if (status || a.rows <= s.rows) return status;
    if (a.merge) {
      const int64_t numbers = a.rows / (kMergeTiles * s.rows);
      const int by_number = numbers < a.segments;
      status = in_launches(a, by_number ? numbers : a.segments, [&](unsigned blocks) {
        gn_merge_kernel<true><<<dim3(blocks, (a.groups + 3) / 4), kThreads, 0, stream>>>(a, means, means + 1, 2, by_number);
      });
      if (status) return status;
    }
    return in_launches(a, second_count(a, s), [&](unsigned blocks) {
      gn_apply_bwd_kernel<T, V, NV, NR><<<dim3(blocks, s.chunks), kThreads, 4 * (s.chunk / a.width) * 4, stream>>>(a, means);
    });
  });
  if (status || !gw) return status;
  return columns<T>(part, tile_count(a, s), a.channels, sums, gw, gb, stream);
}

constexpr int kMostWidth = 8192;

bool sizes_fit(const GnArgs& a) {
  return a.rows >= 1 && a.channels >= 1 && a.groups >= 1 && a.channels % a.groups == 0 && a.width <= kMostWidth && a.segments >= 0 &&
         a.rows < (int64_t(1) << 40) && a.act >= kActNone && a.act <= kActRelu && a.groups <= 65535 * 4;
}

GnArgs arguments(int32_t act, int64_t rows, int32_t channels, int32_t groups, int32_t segments, const int64_t* offsets) {
  GnArgs a{};
  a.act = act;
  a.rows = rows;
  a.channels = channels;
  a.groups = groups;
  a.width = groups > 0 ? channels / groups : 0;
  a.segments = segments;
  a.off = offsets;
  return a;
}

}  // namespace

extern "C" {

int64_t fmd_group_norm_work_size(int32_t bf16, int64_t rows, int32_t channels, int32_t groups, int32_t segments) {
  GnArgs a = arguments(0, rows, channels, groups, segments, nullptr);
  if (!sizes_fit(a) || segments < 1) return 0;
  // the largest number of tiles that any alignment leads to: that of the smallest tile
  a.x_ld = 1;
  int64_t most = 0;
  for (int v = 1; v <= 8; v *= 2) {
    a.x_ld = channels % v == 0 ? v : 1;
    const int64_t n = tile_count(a, tile_shape(a, bf16 ? 2 : 4, false));
    most = n > most ? n : most;
  }
  return 2 * most * groups;
}

int fmd_group_norm(int32_t bf16, int32_t act, const void* x, int64_t x_ld, const void* weight, const void* bias, int64_t rows,
                   int32_t channels, int32_t groups, const int64_t* offsets, int32_t segments, float eps, void* y, float* mean,
                   float* inverse, float* work, hipStream_t stream) {
  GnArgs a = arguments(act, rows, channels, groups, segments, offsets);
  a.x = x;
  a.x_ld = x_ld;
  a.weight = weight;
  a.bias = bias;
  a.eps = eps;
  a.y = y;
  a.mean = mean;
  a.inverse = inverse;
  a.part = work;
  FMD_REQUIRE(sizes_fit(a) && x && y && eps >= 0.f && (!offsets || (mean && inverse && work)));
  return bf16 ? norm<__bf16>(a, stream) : norm<float>(a, stream);
}

int64_t fmd_group_norm_bwd_work_size(int32_t bf16, int64_t rows, int32_t channels, int32_t groups, int32_t segments) {
  GnArgs a = arguments(0, rows, channels, groups, segments, nullptr);
  if (!sizes_fit(a)) return 0;
  const int64_t none = 0;
  if (segments >= 1) a.off = &none;
  int64_t most = 0;
  for (int v = 1; v <= 8; v *= 2) {
    a.x_ld = channels % v == 0 ? v : 1;
    const BackSpace s = back_space(a, bf16 ? 2 : 4);
    const int64_t size = s.columns + s.part + s.means + s.sums;
    most = size > most ? size : most;
  }
  return most;
}

int fmd_group_norm_bwd(int32_t bf16, int32_t act, const void* gy, int64_t gy_ld, const void* x, int64_t x_ld, const void* weight,
                       const void* bias, int64_t rows, int32_t channels, int32_t groups, const int64_t* offsets, int32_t segments,
                       const float* mean, const float* inverse, void* gx, void* g_weight, void* g_bias, float* work,
                       hipStream_t stream) {
  GnArgs a = arguments(act, rows, channels, groups, segments, offsets);
  a.x = x;
  a.x_ld = x_ld;
  a.g = gy;
  a.g_ld = gy_ld;
  a.weight = weight;
  a.bias = bias;
  a.gx = gx;
  a.mean = const_cast<float*>(mean);
  a.inverse = const_cast<float*>(inverse);
  FMD_REQUIRE(sizes_fit(a) && x && gy && gx && mean && inverse && work && (!g_weight || g_bias));
  return bf16 ? norm_bwd<__bf16>(a, work, g_weight, g_bias, stream) : norm_bwd<float>(a, work, g_weight, g_bias, stream);
}

}  // extern "C"
