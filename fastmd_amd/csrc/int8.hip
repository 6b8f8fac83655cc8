// Products with weights held in 8-bit integers: rows are rounded to 8 bits with a scale for each, the product is exact in 32-bit
// integers, and its epilogue multiplies by the row's and the channel's scale.
#include "direct_product.h"

namespace {

// x / scale to the nearest integer; 0 where there is none (scale 0, or not finite: the product is then 0 or NaN by its scale)
__device__ __forceinline__ int8_t to_int8(float x, float scale) {
  const float q = rintf(x / scale);
  return (int8_t)(scale == 0.f || !(fabsf(q) < INFINITY) ? 0.f : fminf(fmaxf(q, -127.f), 127.f));
}

struct Eight {
  float v[8];
};

__device__ __forceinline__ Eight load8(const float* p) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
__device__ __forceinline__ Eight load8(const __bf16* p) {
  const fmd_bf16x8 x = *reinterpret_cast<const fmd_bf16x8*>(p);
  Eight r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.v[e] = (float)x[e];
  return r;
}

struct RowArgs {
  const void* x;
  int64_t x_ld, width, rows;
  int8_t* q;
  int64_t q_ld;  // a multiple of 8
  float* scales;
  int32_t wide;  // rows in whole 16-byte vectors
  int64_t row0;
};

template <typename T>
__device__ __forceinline__ Eight row_part(const RowArgs& a, const T* src, int64_t k) {
  if (a.wide && k + 8 <= a.width) return load8(src + k);
  Eight r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.v[e] = k + e < a.width ? (float)src[k + e] : 0.f;
  return r;
}

__device__ __forceinline__ void put_part(int8_t* q, const Eight& x, float scale) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e / 4] |= (uint32_t)(uint8_t)to_int8(x.v[e], scale) << (8 * (e % 4));
  *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
}

// A wave or (LANES 256) a workgroup a row, in registers: NV vectors of eight a lane; NV 0: read twice, whatever its width. 8 192 rows
// of 4 096, bf16: 71 us with a value at a time, 31 so (3.2 TB/s).
template <typename T, int LANES, int NV>
__global__ void __launch_bounds__(256) quantize_rows_kernel(RowArgs a) {
  __shared__ float lds[4];
  const int lane = threadIdx.x % LANES;
  const int64_t row = a.row0 + (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const bool live = row < a.rows;
  const T* src = static_cast<const T*>(a.x) + (live ? row : 0) * a.x_ld;
  Eight x[NV > 0 ? NV : 1];
  float top = 0.f;
  if constexpr (NV > 0) {
#pragma unroll
    for (int n = 0; n < NV; ++n) x[n] = row_part<T>(a, src, (int64_t)(lane + n * LANES) * 8);
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = nan_max(top, fabsf(x[n].v[e]));
  } else {
    for (int64_t k = lane * 8; k < a.width; k += LANES * 8) {
      x[0] = row_part<T>(a, src, k);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = nan_max(top, fabsf(x[0].v[e]));
    }
  }
  top = wave_nan_max(top);
  if (LANES > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
    __syncthreads();
    top = nan_max(nan_max(lds[0], lds[1]), nan_max(lds[2], lds[3]));
  }
  if (!live) return;
  const float scale = top * (1.f / 127.f);
  if (lane == 0) a.scales[row] = scale;
  int8_t* q = a.q + row * a.q_ld;
  if constexpr (NV > 0) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int64_t k = (int64_t)(lane + n * LANES) * 8;
      if (k < a.q_ld) put_part(q + k, x[n], scale);
    }
  } else {
    for (int64_t k = lane * 8; k < a.q_ld; k += LANES * 8) put_part(q + k, row_part<T>(a, src, k), scale);
  }
}

template <typename T>
int quantize(RowArgs a, hipStream_t stream) {
  a.wide = a.x_ld * sizeof(T) % 16 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
  const int64_t vectors = fmd_cdiv(a.q_ld, 8);
  const int each = vectors <= 128 ? 4 : 1;  // rows of a workgroup
  constexpr int64_t most = 1 << 22;
  for (a.row0 = 0; a.row0 < a.rows; a.row0 += most * each) {
    const int64_t left = fmd_cdiv(a.rows - a.row0, each);
    const unsigned blocks = (unsigned)(left < most ? left : most);
#define QUANTIZE(LANES, NV) quantize_rows_kernel<T, LANES, NV><<<blocks, 256, 0, stream>>>(a)
    if (vectors <= 64)
      QUANTIZE(64, 1);
    else if (vectors <= 128)
      QUANTIZE(64, 2);
    else if (vectors <= 256)
      QUANTIZE(256, 1);
    else if (vectors <= 512)
      QUANTIZE(256, 2);
    else if (vectors <= 1024)
      QUANTIZE(256, 4);
    else
      QUANTIZE(256, 0);
#undef QUANTIZE
    FMD_CHECK_LAUNCH();
  }
  return FMD_OK;
}

// Scales and bias in float64, so that the result is rounded once to float32: a sum of 2^27 times a row's scale can pass the largest float32,
// or a scale near the smallest lose its bits, where the channel's scale brings the result back. 8 192 rows of 4 096 x 4 096, bf16: 177 us with
// the rounding of the rows, as in float32.
struct ScaleEpi {
  void* out;
  const float *row_scale, *col_scale, *bias;
  int64_t rows, cols;
  int32_t bf16;
  typedef TpNothing Fetch;
  __device__ __forceinline__ Fetch fetch(int64_t, int64_t) const { return {}; }
  __device__ __forceinline__ void operator()(int, int64_t m, int64_t n, int4 v, int4, Fetch) const {
    if (m >= rows || n >= cols) return;
    const double s = row_scale[m];
    const int e[4] = {v.x, v.y, v.z, v.w};
    float o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t c = n + k < cols ? n + k : cols - 1;
      o[k] = (float)(e[k] * s * col_scale[c] + (bias ? bias[c] : 0.f));
    }
    if (bf16) {
      __bf16* p = static_cast<__bf16*>(out) + m * cols + n;
      if (cols % 4 == 0) {
        fmd_bf16x4 x;
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = (__bf16)o[k];
        *reinterpret_cast<fmd_bf16x4*>(p) = x;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (n + k < cols) p[k] = (__bf16)o[k];
      }
    } else {
      float* p = static_cast<float*>(out) + m * cols + n;
      if (cols % 4 == 0) {
        *reinterpret_cast<float4*>(p) = make_float4(o[0], o[1], o[2], o[3]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (n + k < cols) p[k] = o[k];
      }
    }
  }
};

typedef TpShape<TpInt8, 2, 4, 4, 2, false, false, false, 2> Large;
typedef TpShape<TpInt8, 2, 2, 2, 2, false, false, false, 2> Middle;
typedef TpShape<TpInt8, 1, 2, 2, 1, false, false, false, 2> Small;

template <typename Fn>
int with_shape(TpArgs& a, const Fn& fn) {
  const int64_t slices = fmd_cdiv(a.p[0].k, kTpSlice);
  const int64_t tiles = tp_tiles<Large>(a.p[0], 0);
  if (tiles > kTpMostTiles) return FMD_EINVAL;
  const TpPlan large = tp_plan<Large>(tiles, slices, 1.f);
  if (tiles >= 1024) return fn(Large{}, large);
  const TpPlan middle = tp_plan<Middle>(tp_tiles<Middle>(a.p[0], 0), slices, 1.f);
  const TpPlan small = tp_plan<Small>(tp_tiles<Small>(a.p[0], 0), slices, 1.f);
  if (small.time < middle.time && small.time < large.time) return fn(Small{}, small);
  if (middle.time < large.time) {
    tp_tiles<Middle>(a.p[0], 0);
    return fn(Middle{}, middle);
  }
  tp_tiles<Large>(a.p[0], 0);
  return fn(Large{}, large);
}

TpArgs arguments(const int8_t* x, int64_t x_ld, const int8_t* w, int64_t w_ld, int64_t rows, int64_t width, int64_t out) {
  TpArgs a{};
  a.p[0] = {tp_operand(w, w, w_ld, 0, 1), tp_operand(x, x, x_ld, 0, 1), out, rows, width, 1, kTpPlain, 0, 0, 0};
  a.count = 1;
  return a;
}

bool sizes_fit(int64_t rows, int64_t width, int64_t out) {
  return rows >= 1 && rows < (int64_t(1) << 31) && out >= 1 && out < (int64_t(1) << 31) && width >= 1 && width < 131072;
}

bool rows_fit(const int8_t* p, int64_t ld, int64_t width) {
  return p && ld >= width && ld % 16 == 0 && ld <= kTpMostLd && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

// bytes of rounded rows and their scales
int64_t rounded_size(int64_t rows, int64_t width) {
  const int64_t ld = (width + 15) & ~int64_t(15);
  return ((rows * ld + 255) & ~int64_t(255)) + ((rows * 4 + 255) & ~int64_t(255));
}

// A small product with small weights: straight from memory (direct_product.h), with nothing to join. us of rounding and product
// in graphs, tiles and straight: 16 rows of 1 024 x 1 024 12.8 12.0, of 2 048 x 2 048 15.5 12.1, of 4 096 x 4 096 16.9 18.2 (eagerly, weights not
// in caches, 18.5 16.8), of 8 192 x 8 192 26.4 37.4; one of 11 008 x 4 096 24.0 30.2; 64 of 2 048 x 2 048 16.8 12.7, of 4 096 x 4 096 17.2 19.6;
// 128 of 1 024 x 1 024 14.1 11.4; 500 of 1 024 x 1 024 14.9 14.3; 2 000 of 512 x 512 12.5 14.3, of 1 024 x 1 024 17.6 28.2.
bool few_rows(int64_t rows, int64_t width, int64_t out) {
  if (fmd_cdiv(rows, 16) * fmd_cdiv(out, 16) >= int64_t(1) << 22) return false;  // one launch
  return (double)rows * width * out <= 4e8 && (double)width * out <= 2.5e7;
}

int product(const int8_t* x, int64_t x_ld, const int8_t* w, int64_t w_ld, int64_t rows, int64_t width, int64_t out, const ScaleEpi& epi,
            void* work, hipStream_t stream) {
  if (few_rows(rows, width, out)) {
    // whole vectors: past the width one of the two is zero, and both can be read
    const int64_t k = (width + 15) & ~int64_t(15);
    const DpArgs a{{{w, w}, w_ld, 0, 1}, {{x, x}, x_ld, 0, 1}, out, rows, k, 1, 0, 0};
    return dp_product<int8_t, false, false, false>(a, epi, stream);
  }
  TpArgs a = arguments(x, x_ld, w, w_ld, rows, width, out);
  return with_shape(a, [&](auto shape, const TpPlan& plan) { return tp_launch<decltype(shape)>(a, plan, work, epi, stream); });
}

}  // namespace

extern "C" {

int fmd_quantize_rows(int32_t bf16, const void* x, int64_t x_ld, int64_t rows, int64_t width, int8_t* values, int64_t values_ld,
                      float* scales, hipStream_t stream) {
  FMD_REQUIRE(rows >= 0 && width >= 1 && values_ld >= width && values_ld % 8 == 0 && (reinterpret_cast<uintptr_t>(values) & 7) == 0 &&
              (rows == 0 || (x && values && scales)));
  const RowArgs a{x, x_ld, width, rows, values, values_ld, scales, 0, 0};
  return bf16 ? quantize<__bf16>(a, stream) : quantize<float>(a, stream);
}

int64_t fmd_linear_int8_work_size(int32_t rounded, int64_t rows, int64_t width, int64_t out) {
  if (!sizes_fit(rows, width, out)) return 0;
  int64_t size = rounded ? 0 : rounded_size(rows, width);
  TpArgs a = arguments(nullptr, 16, nullptr, 16, rows, width, out);
  if (!few_rows(rows, width, out))
    with_shape(a, [&](auto, const TpPlan& plan) {
      size += plan.partial;
      return (int)FMD_OK;
    });
  return size;
}

int fmd_linear_int8(int32_t bf16, const int8_t* x, int64_t x_ld, const float* x_scales, const int8_t* w, int64_t w_ld,
                    const float* w_scales, const float* bias, int64_t rows, int64_t width, int64_t out, void* y, void* work,
                    hipStream_t stream) {
  FMD_REQUIRE(sizes_fit(rows, width, out) && rows_fit(x, x_ld, width) && rows_fit(w, w_ld, width) && x_scales && w_scales && y);
  FMD_REQUIRE(work || !fmd_linear_int8_work_size(1, rows, width, out));
  const ScaleEpi epi{y, x_scales, w_scales, bias, rows, out, bf16};
  return product(x, x_ld, w, w_ld, rows, width, out, epi, work, stream);
}

int fmd_linear_int8_rows(int32_t x_bf16, const void* x, int64_t x_ld, int32_t bf16, const int8_t* w, int64_t w_ld, const float* w_scales,
                         const float* bias, int64_t rows, int64_t width, int64_t out, void* y, void* work, hipStream_t stream) {
  FMD_REQUIRE(sizes_fit(rows, width, out) && x && rows_fit(w, w_ld, width) && w_scales && y && work);
  int8_t* q = static_cast<int8_t*>(work);
  const int64_t q_ld = (width + 15) & ~int64_t(15);
  float* scales = reinterpret_cast<float*>(q + ((rows * q_ld + 255) & ~int64_t(255)));
  const int status = fmd_quantize_rows(x_bf16, x, x_ld, rows, width, q, q_ld, scales, stream);
  if (status) return status;
  const ScaleEpi epi{y, scales, w_scales, bias, rows, out, bf16};
  return product(q, q_ld, w, w_ld, rows, width, out, epi, q + rounded_size(rows, width), stream);
}

}  // extern "C"
