// The gated feed-forward block of small weights in one kernel, forward or backward: a workgroup takes 16 MT rows through all of it,
// the hidden layer (or the gradients of the two projections) stays in LDS, and memory sees the rows alone. Every workgroup reads all
// weights, from the caches. The backward pass forms the projections again: at such widths that is less than writing them and
// reading them back.
//
// For the weights' gradients the backward pass also writes what their products multiply: h, dg and du, in the planes that LDS holds of them
// (float32 three, bf16 two).
#pragma once

#include "activation.h"
#include "direct_product.h"

struct FfnBlock {
  const void *x, *gate, *up, *down, *gy;
  int64_t x_ld, w_ld, d_ld, gy_ld;
  int32_t x_wide, w_wide, d_wide, gy_wide;  // rows in whole 16-byte vectors
  int64_t rows;
  int32_t width, hidden, out, act;
  void* result;     // y [rows, out], or gx [rows, width] (nullable), contiguous
  __bf16 *h, *d;    // backward, nullable: [planes, rows, hp], [planes, 2, rows, hp]
  int64_t hp;
  int64_t row0;     // first row of this launch
};

constexpr int kBlockWaves = 8, kBlockThreads = 64 * kBlockWaves;
constexpr int kBlockLds = 65536;

// row stride in LDS, elements: whole units of K, and eight more so that sixteen rows' chunks fall on different banks
__host__ __device__ inline int block_ld(int hidden) { return (hidden + 31) / 32 * 32 + 8; }
inline int block_lds(int hidden, int planes, int rows, bool back) { return (back ? 2 : 1) * planes * rows * block_ld(hidden) * 2; }

// acc[g][t] += rows of n_op[g] times the rows of m, over K; the n operand along or across K
template <typename T, bool ACROSS, int G, int MT>
__device__ __forceinline__ void block_product(typename DpType<T>::Acc (&acc)[G][MT], const void* const (&n)[G], const DpOperand& on, int64_t row_n,
                                              const void* m, const DpOperand& om, int64_t m0, int64_t rows, int k, int lane) {
  typedef DpType<T> D;
  constexpr int U = sizeof(T) == 4 ? 2 : 4;
  const int r = lane & 15, q = lane >> 4;
  for (int first = 0; first < k; first += U * D::UNIT) {
    DpLoad<T, ACROSS, false> ln[G][U];
    DpLoad<T, false, false> lm[MT][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = first + u * D::UNIT + q * D::EACH;
#pragma unroll
      for (int g = 0; g < G; ++g) ln[g][u].load(on, n[g], row_n, at, k);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int64_t row = m0 + 16 * t + r;
        lm[t][u].load(om, m, row < rows ? row : rows - 1, at, k);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      tp_i32x4 pn[G][D::PLANES], pm[D::PLANES];
#pragma unroll
      for (int g = 0; g < G; ++g) ln[g][u].planes(pn[g]);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        lm[t][u].planes(pm);
#pragma unroll
        for (int g = 0; g < G; ++g) acc[g][t] = dp_mma<T>(pn[g], pm, acc[g][t]);
      }
    }
  }
}

// Four values of an operand in LDS or in memory: the three planes of float32, or two for a product with bf16. Of an infinite value the
// second is zero: its products with finite ones stay infinite.
template <int PLANES>
__device__ __forceinline__ void put_planes(__bf16* p, int64_t plane, const float (&v)[4]) {
  fmd_bf16x4 x[3];
  x3_split(make_float4(v[0], v[1], v[2], v[3]), x[0], x[1], x[2]);
  if (PLANES == 2) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[1][e] = fabsf((float)x[0][e]) == INFINITY ? (__bf16)0.f : x[1][e];
  }
#pragma unroll
  for (int i = 0; i < PLANES; ++i) *reinterpret_cast<fmd_bf16x4*>(p + i * plane) = x[i];
}

template <typename T>
struct RawFour {
  typedef T Type __attribute__((ext_vector_type(4)));
};

template <typename T, int MT, bool BACK>
__global__ void __launch_bounds__(kBlockThreads) ffn_block_kernel(FfnBlock a) {
  typedef DpType<T> D;
  constexpr int ROWS = 16 * MT, P = D::KEPT;
  extern __shared__ __attribute__((aligned(16))) char block_lds_space[];
  __bf16* lds = reinterpret_cast<__bf16*>(block_lds_space);  // [BACK ? dg, du : h][planes][ROWS][ld]
  const int ld = block_ld(a.hidden), plane = ROWS * ld;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
  const int64_t m0 = a.row0 + (int64_t)blockIdx.x * ROWS;
  const DpOperand ox{{a.x, a.x}, a.x_ld, 0, a.x_wide}, og{{a.gy, a.gy}, a.gy_ld, 0, a.gy_wide};
  const DpOperand ow{{a.gate, a.up}, a.w_ld, 0, a.w_wide}, od{{a.down, a.down}, a.d_ld, 0, a.d_wide};

  // sixteen columns of the hidden layer a wave, past the last one zeros up to whole units of K
  for (int n0 = 16 * wave; n0 < ld - 8; n0 += 16 * kBlockWaves) {
    const int64_t row_n = n0 + r < a.hidden ? n0 + r : a.hidden - 1;
    typename D::Acc acc[2][MT], back[1][MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[0][t] = acc[1][t] = back[0][t] = typename D::Acc{0, 0, 0, 0};
    if (n0 < a.hidden) {
      const void* const projections[2] = {a.gate, a.up};
      block_product<T, false, 2, MT>(acc, projections, ow, row_n, a.x, ox, m0, a.rows, a.width, lane);
      if (BACK) {
        const void* const down[1] = {a.down};
        block_product<T, true, 1, MT>(back, down, od, row_n, a.gy, og, m0, a.rows, a.out, lane);
      }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      float h[4], dg[4], du[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = n0 + 4 * q + e < a.hidden;
        const float g = acc[0][t][e], u = acc[1][t][e], gh = back[0][t][e];
        const ActValue v = activation(g, a.act);
        h[e] = in ? v.value * u : 0.f;
        dg[e] = in ? gh * u * v.slope : 0.f;
        du[e] = in ? gh * v.value : 0.f;
      }
      __bf16* to = lds + (16 * t + r) * ld + n0 + 4 * q;
      if (!BACK) {
        put_planes<P>(to, plane, h);
        continue;
      }
      put_planes<P>(to, plane, dg);
      put_planes<P>(to + P * plane, plane, du);
      const int64_t m = m0 + 16 * t + r, n = n0 + 4 * q;
      if (a.d && m < a.rows && n < a.hp) {
        put_planes<P>(a.h + m * a.hp + n, a.rows * a.hp, h);
        put_planes<P>(a.d + m * a.hp + n, 2 * a.rows * a.hp, dg);
        put_planes<P>(a.d + (a.rows + m) * a.hp + n, 2 * a.rows * a.hp, du);
      }
    }
  }
  if (BACK && !a.result) return;
  __syncthreads();

  const int columns = BACK ? a.width : a.out;
  for (int n0 = 16 * wave; n0 < columns; n0 += 16 * kBlockWaves) {
    const int64_t row_n = n0 + r < columns ? n0 + r : columns - 1;
    typename D::Acc acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = typename D::Acc{0, 0, 0, 0};
#pragma unroll
    for (int part = 0; part < (BACK ? 2 : 1); ++part) {
      constexpr int U = sizeof(T) == 4 ? 2 : 4;
      const void* n = BACK ? (part ? a.up : a.gate) : a.down;
      for (int first = 0; first < a.hidden; first += U * D::UNIT) {
        DpLoad<T, BACK, false> ln[U];
#pragma unroll
        for (int u = 0; u < U; ++u) ln[u].load(BACK ? ow : od, n, row_n, first + u * D::UNIT + q * D::EACH, a.hidden);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int k = first + u * D::UNIT + q * D::EACH;
          if (first + u * D::UNIT >= a.hidden) break;
          tp_i32x4 pn[D::PLANES], pm[P];
          ln[u].planes(pn);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
#pragma unroll
            for (int i = 0; i < P; ++i)
              pm[i] = *reinterpret_cast<const tp_i32x4*>(lds + (part * P + i) * plane + (16 * t + r) * ld + k);
            acc[t] = dp_mma<T>(pn, pm, acc[t]);
          }
        }
      }
    }
    const int n = n0 + 4 * q;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int64_t m = m0 + 16 * t + r;
      if (m >= a.rows || n >= columns) continue;
      T* to = static_cast<T*>(a.result) + m * columns + n;
      if (columns % 4 == 0) {
        typename RawFour<T>::Type v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)acc[t][e];
        *reinterpret_cast<typename RawFour<T>::Type*>(to) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < columns) to[e] = (T)acc[t][e];
      }
    }
  }
}
