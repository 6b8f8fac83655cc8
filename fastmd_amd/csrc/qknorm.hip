// Norm of queries and keys over each head with the rotation of the position in the same pass, and its VJP.
//
//   r = (mean x^2 + eps)^(-1/2),  y = x r w,  (a, b) -> (a cos - b sin, b cos + a sin) on the first `rot` columns
//
// A row (one head of one token) belongs to a group of LG lanes, eight columns each: one read, one write, the mean by
// lane exchanges. The angles come from tables, one row for all heads of a token. All arithmetic is fp32, each output rounded
// once. Memory bounds both directions (of a large copy's 4.8 TB/s): 40 000 tokens of 20 heads of 128, bf16, half of the columns
// turned, 84-87 us forward (4.9 TB/s), 192 VJP (3.2); 16 875 tokens of 16 heads of 64, fp32, 27 us (5.1) and 43 (4.9, with the
// weights' gradients); below some 2 000 rows the host's time for a launch does. The bf16 VJP issues as many instructions as its
// loads can hide: units counted in 32 bits instead of 64, and the reciprocal root in one instruction, took 5 % off it.
#include "attention.h"

namespace {

// The forward takes four heads of a token in a unit: their loads are in flight together and the token's angles and weights are
// read once (16 875 x 16 x 64 fp32 27.3 us, of two 26.9, of eight 26.0; 40 000 x 20 x 128 bf16 86, 88, 83; 40 000 x 3 x 256
// 39, -, 60; 100 000 x 8 x 32 fp32 38, -, 42). The VJP, which holds twice as much of each, takes one: 44 us in the first
// of these against 54 of two and 52 of four, 208 against 250 of two in the second, 58 against 74, 73 against 92.
constexpr int kFwdHeads = 4;

struct NormArgs {
  const void *q, *k;  // [tokens, heads, dim]; k may be null
  int64_t q_row, q_head, k_row, k_head;
  int32_t heads, kv_heads, dim, rot, interleaved, norm;
  int64_t tokens;
  float eps;
  const void *wq, *wk;     // [dim] or null (ones)
  const float *cs, *sn;    // tables [table_rows, rot / 2]
  int64_t table_rows, table_ld;
  const void* positions;   // null: token t takes table row t
  int32_t pos64;
};

template <int LG>
__device__ __forceinline__ float group_sum(float x) {
  x = lanes_sum<(LG < 16 ? LG : 16)>(x);
  if (LG == 32) {
    float y = x;
    swap_halves16(x, y);
    x += y;
  }
  return x;
}

// How the other column of a pair is reached: neighbours of a lane; the same place of another lane of the group (rot / 2 a
// multiple of eight); anywhere, by eight exchanges a column, which then bound it (16 875 tokens of 16 heads of 64, fp32, 20 columns
// turned 40 us forward and 62 VJP, 64 columns 27 and 43; 40 000 of 20 heads of 128, bf16, 40 columns 139 and 273, 64 neighbouring 84 and 194).
enum Turn { kNone, kNeighbours, kLanes, kAnywhere };

__device__ __forceinline__ int64_t table_row(const NormArgs& a, int64_t tok) {
  const int64_t p = !a.positions ? tok
                    : a.pos64    ? static_cast<const int64_t*>(a.positions)[tok]
                                 : static_cast<const int32_t*>(a.positions)[tok];
  return p >= 0 && p < a.table_rows ? p : -1;
}

// cosine and sine of each of the lane's columns (1 and 0 past `rot`; NaN for a position outside the table)
template <Turn TURN>
__device__ __forceinline__ void angles(const NormArgs& a, int64_t tok, int col0, float (&c)[8], float (&s)[8]) {
  if constexpr (TURN == kNone) return;
  const int64_t p = table_row(a, tok);
  const int half = a.rot >> 1;
  const float *cs = a.cs + p * a.table_ld, *sn = a.sn + p * a.table_ld;
  if (TURN == kNeighbours && col0 + 8 <= a.rot && p >= 0 && (a.table_ld & 3) == 0) {  // four angles in a row
    const float4 x = *reinterpret_cast<const float4*>(cs + (col0 >> 1));
    const float4 y = *reinterpret_cast<const float4*>(sn + (col0 >> 1));
    c[0] = c[1] = x.x, c[2] = c[3] = x.y, c[4] = c[5] = x.z, c[6] = c[7] = x.w;
    s[0] = s[1] = y.x, s[2] = s[3] = y.y, s[4] = s[5] = y.z, s[6] = s[7] = y.w;
    return;
  }
  if (TURN == kLanes && p >= 0 && (a.table_ld & 3) == 0) {  // eight
    if (col0 >= a.rot) return;
    load8<float>(cs + (col0 < half ? col0 : col0 - half), c);
    load8<float>(sn + (col0 < half ? col0 : col0 - half), s);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int col = col0 + e, i = TURN == kNeighbours ? col >> 1 : col < half ? col : col - half;
    if (col < a.rot) {
      c[e] = p >= 0 ? cs[i] : NAN;
      s[e] = p >= 0 ? sn[i] : NAN;
    }
  }
}

// y -> rotated y (sign 1) or the transposed rotation (sign -1). Columns past `rot` stay as they are, whatever they hold (a product
// with a sine of zero would make NaN of an infinity, and of a NaN beside them).
template <int LG, Turn TURN>
__device__ __forceinline__ void rotate(const NormArgs& a, int col0, const float (&c)[8], const float (&s)[8], float sign,
                                       float (&y)[8]) {
  if constexpr (TURN == kNone) return;
  const int half = a.rot >> 1;
  float o[8];
  if constexpr (TURN == kNeighbours) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const bool turned = col0 + e < a.rot;
      o[e] = turned ? y[e] * c[e] - sign * s[e] * y[e + 1] : y[e];
      o[e + 1] = turned ? y[e + 1] * c[e + 1] + sign * s[e + 1] * y[e] : y[e + 1];
    }
  } else if constexpr (TURN == kLanes) {
    const int lane = threadIdx.x & 63, sub = lane & (LG - 1), by = half >> 3;
    const bool low = col0 < half;
    const int from = (lane - sub) + (col0 < a.rot ? (low ? sub + by : sub - by) : sub);
    const float f = low ? -sign : sign;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float other = __shfl(y[e], from, 64);
      o[e] = col0 < a.rot ? y[e] * c[e] + f * s[e] * other : y[e];
    }
  } else {
    const int lane = threadIdx.x & 63, base = lane & ~(LG - 1);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int col = col0 + e;
      const int other = col < half ? col + half : col < a.rot ? col - half : col;
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {  // the lane that holds `other`, at each of its places
        const float x = __shfl(y[k], base + (other >> 3), 64);
        v = (other & 7) == k ? x : v;
      }
      o[e] = col < a.rot ? y[e] * c[e] + (col < half ? -sign : sign) * s[e] * v : y[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = o[e];
}

// the units of work of the whole call: (token, block of `by` heads), queries and keys in blocks of their own
__device__ __forceinline__ int head_blocks(const NormArgs& a, int by) {
  return (a.heads + by - 1) / by + (a.kv_heads + by - 1) / by;
}

template <typename T, int LG, Turn TURN, bool NT>
__global__ void __launch_bounds__(256) qk_norm_kernel(NormArgs a, uint32_t block0, T* q_out, T* k_out) {
  const int sub = threadIdx.x & (LG - 1), col0 = 8 * sub;
  const uint32_t unit = (block0 + blockIdx.x) * (256 / LG) + threadIdx.x / LG;  // fewer than 2^31 of them
  const int blocks = head_blocks(a, kFwdHeads), qb = (a.heads + kFwdHeads - 1) / kFwdHeads;
  int64_t tok = unit / (uint32_t)blocks;
  const int hb = (int)(unit % (uint32_t)blocks);
  const bool in = tok < a.tokens, is_k = hb >= qb;
  if (!in) tok = 0;
  const int h0 = (is_k ? hb - qb : hb) * kFwdHeads, heads = is_k ? a.kv_heads : a.heads;
  const T* x = static_cast<const T*>(is_k ? a.k : a.q) + tok * (is_k ? a.k_row : a.q_row);
  const int64_t hs = is_k ? a.k_head : a.q_head;
  T* out = (is_k ? k_out : q_out) + tok * heads * a.dim;
  const bool cols = col0 < a.dim;
  const float inv_dim = 1.f / a.dim;
  float y[kFwdHeads][8];
#pragma unroll
  for (int h = 0; h < kFwdHeads; ++h) {
    if (in && cols && h0 + h < heads) load8<T>(x + (h0 + h) * hs + col0, y[h]);
    else
#pragma unroll
      for (int e = 0; e < 8; ++e) y[h][e] = 0.f;
  }
  float w[8], c[8], s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = 1.f, c[e] = 1.f, s[e] = 0.f;
  const T* wp = static_cast<const T*>(is_k ? a.wk : a.wq);
  if (cols && wp) load8<T>(wp + col0, w);
  if (in && cols) angles<TURN>(a, tok, col0, c, s);
#pragma unroll
  for (int h = 0; h < kFwdHeads; ++h) {
    if (a.norm) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += y[h][e] * y[h][e];
      const float r = rsqrtf(fmaf(group_sum<LG>(ss), inv_dim, a.eps));
#pragma unroll
      for (int e = 0; e < 8; ++e) y[h][e] = y[h][e] * r * w[e];
    }
    rotate<LG, TURN>(a, col0, c, s, 1.f, y[h]);
    if (in && cols && h0 + h < heads) store8<NT>(out + (h0 + h) * a.dim + col0, y[h]);
  }
}

struct NormGrad {
  const void *gq, *gk;
  int64_t gq_row, gq_head, gk_row, gk_head;
};

// A workgroup takes `per` consecutive units per group; its weight gradients are summed over them in registers, over its
// groups in LDS in order, and written as one row per workgroup, which norm_weights_kernel adds in order.
template <typename T, int LG, Turn TURN, bool NT>
__global__ void __launch_bounds__(256) qk_norm_bwd_kernel(NormArgs a, NormGrad g, int per, T* gq_out, T* gk_out, float* part) {
  constexpr int GROUPS = 256 / LG;
  __shared__ float sum[2][256][8];
  const int sub = threadIdx.x & (LG - 1), col0 = 8 * sub, group = threadIdx.x / LG;
  const uint32_t blocks = a.heads + a.kv_heads, units = (uint32_t)a.tokens * blocks;  // a unit: one head of one token; below 2^31
  const bool cols = col0 < a.dim;
  const float inv_dim = 1.f / a.dim;
  float gw[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) gw[0][e] = gw[1][e] = 0.f;
  for (int n = 0; n < per; ++n) {
    const uint32_t unit = (blockIdx.x * per + n) * GROUPS + group;
    const bool in = unit < units;
    const int64_t tok = in ? unit / blocks : 0;
    const int hb = in ? (int)(unit % blocks) : 0;
    const bool is_k = hb >= a.heads;
    const int h = is_k ? hb - a.heads : hb;
    const T* xp = static_cast<const T*>(is_k ? a.k : a.q) + tok * (is_k ? a.k_row : a.q_row) + h * (is_k ? a.k_head : a.q_head);
    const T* gp = static_cast<const T*>(is_k ? g.gk : g.gq) + tok * (is_k ? g.gk_row : g.gq_row) +
                  h * (is_k ? g.gk_head : g.gq_head);
    T* out = (is_k ? gk_out : gq_out) + (tok * (is_k ? a.kv_heads : a.heads) + h) * a.dim;
    float x[8], y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = y[e] = 0.f;
    if (in && cols) {
      load8<T>(gp + col0, y);
      if (a.norm) load8<T>(xp + col0, x);
    }
    float w[8], c[8], s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.f, c[e] = 1.f, s[e] = 0.f;
    const T* wp = static_cast<const T*>(is_k ? a.wk : a.wq);
    if (cols && wp) load8<T>(wp + col0, w);
    if (in && cols) angles<TURN>(a, tok, col0, c, s);
    rotate<LG, TURN>(a, col0, c, s, -1.f, y);
    if (a.norm) {
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
      const float r = rsqrtf(fmaf(group_sum<LG>(ss), inv_dim, a.eps));
      float gn[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] *= r;  // the normalised value
        gn[e] = y[e] * w[e];
        dot += gn[e] * x[e];
        const float t = y[e] * x[e];
        gw[0][e] += is_k ? 0.f : t;
        gw[1][e] += is_k ? t : 0.f;
      }
      const float mean = group_sum<LG>(dot) * inv_dim;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = r * (gn[e] - x[e] * mean);
    }
    if (in && cols) store8<NT>(out + col0, y);
  }
  if (!part) return;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[k][threadIdx.x][e] = gw[k][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.dim; i += 256) {
    const int k = i / a.dim, col = i % a.dim;
    float t = 0.f;
    for (int n = 0; n < GROUPS; ++n) t += sum[k][n * LG + (col >> 3)][col & 7];
    part[(int64_t)blockIdx.x * 2 * a.dim + i] = t;
  }
}

// gradient of the weights: column sums of the workgroups' rows: 16 columns a workgroup, 64 threads each over every 64th row, joined in order
template <typename T>
__global__ void __launch_bounds__(1024) norm_weights_kernel(const float* part, int rows, int dim, T* gwq, T* gwk) {
  __shared__ float sum[64][16];
  const int col = blockIdx.x * 16 + (threadIdx.x & 15), lane = threadIdx.x >> 4;
  float t = 0.f;
  if (col < 2 * dim)
    for (int r = lane; r < rows; r += 64) t += part[(int64_t)r * 2 * dim + col];
  sum[lane][threadIdx.x & 15] = t;
  __syncthreads();
  for (int n = 32; n >= 1; n >>= 1) {
    if (lane < n) sum[lane][threadIdx.x & 15] += sum[lane + n][threadIdx.x & 15];
    __syncthreads();
  }
  if (lane == 0 && col < 2 * dim) {
    T* out = col < dim ? gwq : gwk;
    if (out) out[col < dim ? col : col - dim] = (T)sum[0][threadIdx.x & 15];
  }
}

int groups_of(int dim) {
  int lg = 1;
  while (8 * lg < dim) lg *= 2;
  return lg;
}

int64_t unit_count(int64_t tokens, int heads, int kv_heads, int by) {
  return tokens * ((heads + by - 1) / by + (kv_heads + by - 1) / by);
}

// workgroups of the VJP: at most 1 024 (four per CU), so that the partial sums stay few (at most 2 048: 49 us against 44 and 215
// against 207 in the cases above)
void bwd_grid(int64_t units, int groups, int* grid, int* per) {
  const int64_t n = fmd_cdiv(units, groups);
  *per = n > 1024 ? (int)fmd_cdiv(n, 1024) : 1;
  *grid = (int)fmd_cdiv(n, *per);
}

bool ok16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
int check_norm(const NormArgs& a) {
  FMD_REQUIRE(a.tokens >= 0 && a.heads >= 0 && a.kv_heads >= 0 && a.heads + a.kv_heads > 0 && a.dim > 0);
  if (a.dim % 8 != 0 || a.dim > 256) return FMD_EUNSUPPORTED;
  FMD_REQUIRE(a.rot >= 0 && a.rot % 2 == 0 && a.rot <= a.dim);
  FMD_REQUIRE(a.tokens == 0 || ((a.heads == 0 || a.q) && (a.kv_heads == 0 || a.k)));
  FMD_REQUIRE(a.rot == 0 || (a.cs && a.sn && a.table_ld >= a.rot / 2 && ok16(a.cs) && ok16(a.sn)));
  FMD_REQUIRE(a.positions || a.rot == 0 || a.table_rows >= a.tokens);
  const int64_t unit = 16 / sizeof(T);
  FMD_REQUIRE(ok16(a.q) && ok16(a.k) && ok16(a.wq) && ok16(a.wk));
  FMD_REQUIRE(a.q_row % unit == 0 && a.q_head % unit == 0 && a.k_row % unit == 0 && a.k_head % unit == 0);
  FMD_REQUIRE(unit_count(a.tokens, a.heads, a.kv_heads, 1) < (1ll << 31));
  return FMD_OK;
}

Turn turn_of(const NormArgs& a) {
  return a.rot == 0 ? kNone : a.interleaved ? kNeighbours : a.rot % 16 == 0 ? kLanes : kAnywhere;
}

template <typename T>
bool streams(const NormArgs& a) {
  return a.tokens * (a.heads + a.kv_heads) * a.dim * (int64_t)sizeof(T) >= kStreamBytes;
}

template <typename T, int LG, Turn TURN>
int norm_fwd_turn(const NormArgs& a, T* q_out, T* k_out, hipStream_t stream) {
  return launch_ranges(fmd_cdiv(unit_count(a.tokens, a.heads, a.kv_heads, kFwdHeads), 256 / LG), [&](unsigned n, int64_t first) {
    if (streams<T>(a)) qk_norm_kernel<T, LG, TURN, true><<<n, 256, 0, stream>>>(a, (uint32_t)first, q_out, k_out);
    else qk_norm_kernel<T, LG, TURN, false><<<n, 256, 0, stream>>>(a, (uint32_t)first, q_out, k_out);
  });
}

template <typename T, int LG>
int norm_fwd(const NormArgs& a, T* q_out, T* k_out, hipStream_t stream) {
  switch (turn_of(a)) {
    case kNone: return norm_fwd_turn<T, LG, kNone>(a, q_out, k_out, stream);
    case kNeighbours: return norm_fwd_turn<T, LG, kNeighbours>(a, q_out, k_out, stream);
    case kLanes: return norm_fwd_turn<T, LG, kLanes>(a, q_out, k_out, stream);
    default: return norm_fwd_turn<T, LG, kAnywhere>(a, q_out, k_out, stream);
  }
}

template <typename T, int LG, Turn TURN>
void norm_bwd_turn(const NormArgs& a, const NormGrad& g, int grid, int per, T* gq, T* gk, float* work, hipStream_t stream) {
  if (streams<T>(a)) qk_norm_bwd_kernel<T, LG, TURN, true><<<grid, 256, 0, stream>>>(a, g, per, gq, gk, work);
  else qk_norm_bwd_kernel<T, LG, TURN, false><<<grid, 256, 0, stream>>>(a, g, per, gq, gk, work);
}

template <typename T, int LG>
int norm_bwd(const NormArgs& a, const NormGrad& g, T* gq, T* gk, T* gwq, T* gwk, float* work, hipStream_t stream) {
  const int64_t units = unit_count(a.tokens, a.heads, a.kv_heads, 1);
  const bool weights = gwq || gwk;
  int grid = 0, per = 0;
  bwd_grid(units, 256 / LG, &grid, &per);
  if (grid > 0) {
    float* part = weights ? work : nullptr;
    switch (turn_of(a)) {
      case kNone: norm_bwd_turn<T, LG, kNone>(a, g, grid, per, gq, gk, part, stream); break;
      case kNeighbours: norm_bwd_turn<T, LG, kNeighbours>(a, g, grid, per, gq, gk, part, stream); break;
      case kLanes: norm_bwd_turn<T, LG, kLanes>(a, g, grid, per, gq, gk, part, stream); break;
      default: norm_bwd_turn<T, LG, kAnywhere>(a, g, grid, per, gq, gk, part, stream);
    }
    FMD_CHECK_LAUNCH();
  }
  if (weights) {
    norm_weights_kernel<T><<<(unsigned)fmd_cdiv(2 * a.dim, 16), 1024, 0, stream>>>(work, grid, a.dim, gwq, gwk);
    FMD_CHECK_LAUNCH();
  }
  return FMD_OK;
}

#define FMD_BY_GROUP(F, ...)                             \
  switch (groups_of(a.dim)) {                            \
    case 1: return F<T, 1>(__VA_ARGS__);                 \
    case 2: return F<T, 2>(__VA_ARGS__);                 \
    case 4: return F<T, 4>(__VA_ARGS__);                 \
    case 8: return F<T, 8>(__VA_ARGS__);                 \
    case 16: return F<T, 16>(__VA_ARGS__);               \
    default: return F<T, 32>(__VA_ARGS__);               \
  }

template <typename T>
int forward(const NormArgs& a, T* q_out, T* k_out, hipStream_t stream) {
  const int status = check_norm<T>(a);
  if (status != FMD_OK) return status;
  if (a.tokens == 0) return FMD_OK;
  FMD_REQUIRE((a.heads == 0 || q_out) && (a.kv_heads == 0 || k_out) && ok16(q_out) && ok16(k_out));
  FMD_BY_GROUP(norm_fwd, a, q_out, k_out, stream)
}

template <typename T>
int backward(const NormArgs& a, const NormGrad& g, T* gq, T* gk, T* gwq, T* gwk, float* work, hipStream_t stream) {
  const int status = check_norm<T>(a);
  if (status != FMD_OK) return status;
  const int64_t unit = 16 / sizeof(T);
  FMD_REQUIRE(a.tokens == 0 || ((a.heads == 0 || (g.gq && gq)) && (a.kv_heads == 0 || (g.gk && gk))));
  FMD_REQUIRE(ok16(g.gq) && ok16(g.gk) && ok16(gq) && ok16(gk));
  FMD_REQUIRE(g.gq_row % unit == 0 && g.gq_head % unit == 0 && g.gk_row % unit == 0 && g.gk_head % unit == 0);
  FMD_REQUIRE(!(gwq || gwk) || (work && a.norm));
  FMD_BY_GROUP(norm_bwd, a, g, gq, gk, gwq, gwk, work, stream)
}

}  // namespace

extern "C" {

#define FMD_NORM_PARAMS                                                                                             \
  const void *q, int64_t q_row, int64_t q_head, int32_t heads, const void *k, int64_t k_row, int64_t k_head,        \
      int32_t kv_heads, int64_t tokens, int32_t dim, int32_t norm, float eps, const void *q_weight,                 \
      const void *k_weight, const float *cos_table, const float *sin_table, int64_t table_rows, int64_t table_ld,   \
      int32_t rot, int32_t interleaved, const void *positions, int32_t positions64
#define FMD_NORM_ARGS                                                                                               \
  {                                                                                                                 \
    q, k, q_row, q_head, k_row, k_head, heads, kv_heads, dim, rot, interleaved, norm, tokens, eps, q_weight,        \
        k_weight, cos_table, sin_table, table_rows, table_ld, positions, positions64                                \
  }

int fmd_qk_norm_rotary(int32_t bf16, FMD_NORM_PARAMS, void* q_out, void* k_out, hipStream_t stream) {
  const NormArgs a = FMD_NORM_ARGS;
  return bf16 ? forward(a, static_cast<__bf16*>(q_out), static_cast<__bf16*>(k_out), stream)
              : forward(a, static_cast<float*>(q_out), static_cast<float*>(k_out), stream);
}

int64_t fmd_qk_norm_rotary_work_size(int64_t tokens, int32_t heads, int32_t kv_heads, int32_t dim) {
  if (tokens <= 0 || heads < 0 || kv_heads < 0 || dim <= 0 || dim > 256) return 0;
  int grid = 0, per = 0;
  bwd_grid(unit_count(tokens, heads, kv_heads, 1), 256 / groups_of(dim), &grid, &per);
  return (int64_t)grid * 2 * dim;
}

int fmd_qk_norm_rotary_bwd(int32_t bf16, FMD_NORM_PARAMS, const void* gq_out, int64_t gq_row, int64_t gq_head,
                           const void* gk_out, int64_t gk_row, int64_t gk_head, void* gq, void* gk, void* gq_weight,
                           void* gk_weight, float* work, hipStream_t stream) {
  const NormArgs a = FMD_NORM_ARGS;
  const NormGrad g = {gq_out, gk_out, gq_row, gq_head, gk_row, gk_head};
  return bf16 ? backward(a, g, static_cast<__bf16*>(gq), static_cast<__bf16*>(gk), static_cast<__bf16*>(gq_weight),
                         static_cast<__bf16*>(gk_weight), work, stream)
              : backward(a, g, static_cast<float*>(gq), static_cast<float*>(gk), static_cast<float*>(gq_weight),
                         static_cast<float*>(gk_weight), work, stream);
}

}  // extern "C"
