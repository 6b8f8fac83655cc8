// Products with weights held in 8-bit integers: rows are rounded to 8 bits with a scale for each, the product is exact in 32-bit
// integers, and its epilogue multiplies by the row's and the channel's scale.
#include "tile_product.h"

namespace {

template <typename T>
__device__ __forceinline__ float value_of(const void* x, int64_t i) {
  return (float)static_cast<const T*>(x)[i];
}

// x / scale to the nearest integer; 0 where there is none (scale 0, or not finite: the product is then 0 or NaN by its scale)
__device__ __forceinline__ int8_t to_int8(float x, float scale) {
  const float q = rintf(x / scale);
  return (int8_t)(scale == 0.f || !(fabsf(q) < INFINITY) ? 0.f : fminf(fmaxf(q, -127.f), 127.f));
}

// One workgroup a row, which it reads twice (the second time from the cache).
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void* x, int64_t x_ld, int64_t width, int8_t* q, int64_t q_ld,
                                                            float* scales, int64_t row0) {
  __shared__ float lds[4];
  const int64_t row = row0 + blockIdx.x;
  const T* src = static_cast<const T*>(x) + row * x_ld;
  float top = 0.f;
  for (int64_t k = threadIdx.x; k < width; k += 256) top = nan_max(top, fabsf((float)src[k]));
  top = wave_nan_max(top);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
  __syncthreads();
  const float scale = nan_max(nan_max(lds[0], lds[1]), nan_max(lds[2], lds[3])) * (1.f / 127.f);
  if (threadIdx.x == 0) scales[row] = scale;
  for (int64_t k = threadIdx.x; k < q_ld; k += 256) q[row * q_ld + k] = k < width ? to_int8((float)src[k], scale) : 0;
}

struct ScaleEpi {
  void* out;
  const float *row_scale, *col_scale, *bias;
  int64_t rows, cols;
  int32_t bf16;
  __device__ __forceinline__ void operator()(int, int64_t m, int64_t n, int4 v, int4) const {
    if (m >= rows || n >= cols) return;
    const float s = row_scale[m];
    const int e[4] = {v.x, v.y, v.z, v.w};
    float o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t c = n + k < cols ? n + k : cols - 1;
      o[k] = (float)e[k] * s * col_scale[c] + (bias ? bias[c] : 0.f);
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
  int64_t tiles = tp_tiles<Large>(a.p[0], 0);
  if (tiles > kTpMostTiles) return FMD_EINVAL;
  if (tiles >= 192) return fn(Large{}, tp_plan<Large>(tiles, slices));
  tiles = tp_tiles<Middle>(a.p[0], 0);
  if (tiles >= 256) return fn(Middle{}, tp_plan<Middle>(tiles, slices));
  tiles = tp_tiles<Small>(a.p[0], 0);
  return fn(Small{}, tp_plan<Small>(tiles, slices));
}

TpArgs arguments(const int8_t* x, int64_t x_ld, const int8_t* w, int64_t w_ld, int64_t rows, int64_t width, int64_t out) {
  TpArgs a{};
  a.p[0] = {tp_operand(w, w, w_ld, 0, 1), tp_operand(x, x, x_ld, 0, 1), out, rows, width, 1, 1, 0, 0, 0};
  a.count = 1;
  return a;
}

bool sizes_fit(int64_t rows, int64_t width, int64_t out) {
  return rows >= 1 && rows < (int64_t(1) << 31) && out >= 1 && out < (int64_t(1) << 31) && width >= 1 && width < 131072;
}

bool rows_fit(const int8_t* p, int64_t ld, int64_t width) {
  return p && ld >= width && ld % 16 == 0 && ld <= kTpMostLd && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

}  // namespace

extern "C" {

int fmd_quantize_rows(int32_t bf16, const void* x, int64_t x_ld, int64_t rows, int64_t width, int8_t* values, int64_t values_ld,
                      float* scales, hipStream_t stream) {
  FMD_REQUIRE(rows >= 0 && width >= 1 && values_ld >= width && (rows == 0 || (x && values && scales)));
  constexpr int64_t most = 1 << 22;
  for (int64_t r = 0; r < rows; r += most) {
    const unsigned blocks = (unsigned)(rows - r < most ? rows - r : most);
    if (bf16)
      quantize_rows_kernel<__bf16><<<blocks, 256, 0, stream>>>(x, x_ld, width, values, values_ld, scales, r);
    else
      quantize_rows_kernel<float><<<blocks, 256, 0, stream>>>(x, x_ld, width, values, values_ld, scales, r);
    FMD_CHECK_LAUNCH();
  }
  return FMD_OK;
}

int64_t fmd_linear_int8_work_size(int64_t rows, int64_t width, int64_t out) {
  if (!sizes_fit(rows, width, out)) return 0;
  TpArgs a = arguments(nullptr, 16, nullptr, 16, rows, width, out);
  int64_t size = 0;
  with_shape(a, [&](auto, const TpPlan& plan) {
    size = plan.partial;
    return (int)FMD_OK;
  });
  return size;
}

int fmd_linear_int8(int32_t bf16, const int8_t* x, int64_t x_ld, const float* x_scales, const int8_t* w, int64_t w_ld,
                    const float* w_scales, const float* bias, int64_t rows, int64_t width, int64_t out, void* y, void* work,
                    hipStream_t stream) {
  FMD_REQUIRE(sizes_fit(rows, width, out) && rows_fit(x, x_ld, width) && rows_fit(w, w_ld, width) && x_scales && w_scales && y && work);
  TpArgs a = arguments(x, x_ld, w, w_ld, rows, width, out);
  const ScaleEpi epi{y, x_scales, w_scales, bias, rows, out, bf16};
  return with_shape(a, [&](auto shape, const TpPlan& plan) { return tp_launch<decltype(shape)>(a, plan, work, epi, stream); });
}

}  // extern "C"
