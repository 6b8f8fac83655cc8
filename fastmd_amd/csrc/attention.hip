// Attention of the query rows of each segment over the key rows of the same segment, and its VJP.
#include <algorithm>
#include <type_traits>

#include "attention.h"

namespace {

// With scores s_ij = scale q_i . k_j over the keys j that query i sees,
//   p_ij = exp(s_ij - max) / sum,   out_i = sum_j p_ij v_j
//   VJP of g: delta_i = g_i . out_i,  gv_j = sum_i p_ij g_i,  ds_ij = scale p_ij (g_i . v_j - delta_i),
//             gq_i = sum_j ds_ij k_j,  gk_j = sum_i ds_ij q_i
// Work: 4 D operations per pair and head forward; 8 D for gk and gv (scores and g . v formed again, two products) and 6 D for gq,
// in two walks: one walk would need atomics, or the sums of one side in memory. Bytes: every row once.

// Waves per SIMD that a kernel is compiled for. Two leave 256 registers, which the compiler then uses as one file; with
// one it puts the sums into accumulation registers and moves them out and back at every rescaling.
static constexpr int attn_waves(int planes, int dp, int sums) { return planes * dp * sums <= 192 ? 2 : 1; }

// bf16 weights (P, dS) are two bf16 parts, the second what the rounding of the first dropped (16 bits together): a product more
// of two forward, of three for gq and two more of four for gk and gv. With one part the rounding of the weights is as large as that of the
// result, however many keys a row has (the terms' errors and the terms add up alike), and the results were 1.4 times as far from
// the exact ones as those rounded once; with two they are as near. It costs, on one card, 287 -> 396 us at 10 000 rows of 8 heads of
// 64, 247 -> 329 in prompts of 12 000 causal rows of 16 heads of 128, 495 -> 608 forward and VJP of 8 192 such rows; where memory bounds,
// nothing.
template <int NP>
__device__ __forceinline__ Planes<NP> rest_of(const float (&x)[8], const Planes<NP>& first) {
  const uint4 w = __builtin_bit_cast(uint4, first.p[0]);  // the parts as they lie in pairs: unpacked, not converted one by one again
  const uint32_t pair[4] = {w.x, w.y, w.z, w.w};
  float y[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[2 * e] = x[2 * e] - __uint_as_float(pair[e] << 16);
    y[2 * e + 1] = x[2 * e + 1] - __uint_as_float(pair[e] & 0xffff0000u);
  }
  Planes<NP> o;
  planes_of(y, o);
  return o;
}

// ------------------------------------------------------------------------------------ forward

// One workgroup: 32 WM packed query rows of one key head, WM KW waves. Wave (wm, kw) holds 32 rows and walks the key
// tiles kw, kw + KW, ... of its split; the KW partial softmaxes are joined through LDS at the end. The scores are
// formed transposed, S^T = K Q^T (lane: a query, registers: keys), so the softmax statistics are one value per lane, the
// sums over keys stay in the lane but for one exchange of the halves, and exp(S^T) is already the operand of
// O^T = V^T P^T. Statistics and sums are fp32; P is kept in two bf16 parts for bf16 inputs and as three planes
// for fp32.
// Measured: bf16, 10 000 rows, 8 heads of 64: 396-404 us, 510 TFLOP/s of the 4 D operations, 770 with the second part's (a large
// library product 1 125): the matrix pipes are busy 40 % of the time, the vector ones with the exponentials (quarter rate), their
// arguments, maxima, sums and parts for most of the rest, and waves of a SIMD overlap the two in part. 5 prompts of 12 000 causal rows
// together, 16 heads of 128: 329-341 us, 630 TFLOP/s (940). fp32, 16 systems of 16 875 rows, 4 heads of 32: 95-103 us, 120 TFLOP/s (the
// library's fp32 154; six bf16 products each, and as much again for splitting P). One query each over 16 x 40 000 keys, 4 heads of 128,
// bf16: 235 us, 5.6 TB/s, memory.
template <typename T, int DP, int BN, int WM, int KW, bool DMA, bool CAUSAL>
__global__ void __launch_bounds__(64 * WM * KW, attn_waves(AttnType<T>::planes, DP, 1)) attn_fwd_kernel(AttnArgs a, AttnTiles kv,
                                                                int64_t tiles, int splits, T* out, AttnSaved saved,
                                                                float* part_o, float* part_m, float* part_l) {
  constexpr int NP = AttnType<T>::planes, DB = DP / 32, KS = DP / 16, JB = BN / 32;
  constexpr bool kTwoParts = NP == 1;
  using Tile = AttnTile<NP, BN, DP>;
  constexpr int kMerge = (KW - 1) * WM * (DB * 16 + 2) * 64 * 2;  // in bf16 units
  constexpr int kTiles = 2 * KW * Tile::SIZE;
  // DMA: tiles of bf16 (or of planes) are copied straight into LDS, a tile ahead, into two buffers; else fp32 tiles go through
  // registers, where they are split, into one
  __shared__ __attribute__((aligned(16))) __bf16 lds[kTiles > kMerge ? kTiles : kMerge];
  __shared__ __attribute__((aligned(16))) __bf16 lds2[DMA ? kTiles : 8];

  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, kw = wave / WM;
  const uint32_t block = a.block0 + blockIdx.x;
  const int kvh = block % a.kv_heads;
  int64_t t = block / a.kv_heads;
  if (CAUSAL) t = tiles - 1 - t;  // the rows with the most keys first
  int64_t first;
  const int ext = attn_find(a.q_off, a.segments, a.tq, a.group, 32 * WM, t, &first, WaveLanes());
  AttnSegment sg = attn_segment(a, ext);
  if (!attn_real(a, ext)) sg.nk = 0;
  const int rows = sg.nq * a.group;
  if (first >= rows) return;
  const int row0 = (int)first, row = row0 + 32 * wm + (lane & 31);
  const bool live = row < rows;
  const int tok = attn_token(a, live ? row : rows - 1), head = kvh * a.group + (live ? row : rows - 1) - tok * a.group;
  const int64_t qt = sg.q0 + tok;

  // keys that this row sees, and that any row of the workgroup sees
  const int shift = sg.nk - sg.nq;
  const int sees = CAUSAL ? max(0, min(sg.nk, tok + shift + 1)) : sg.nk;
  const int last_row = min(row0 + 32 * WM, rows) - 1;
  const int reach = CAUSAL ? max(0, min(sg.nk, attn_token(a, last_row) + shift + 1)) : sg.nk;
  const int least = CAUSAL ? max(0, min(sg.nk, attn_token(a, row0) + shift + 1)) : sg.nk;
  const int all_tiles = (reach + BN - 1) / BN;
  const int per = (all_tiles + splits - 1) / splits;
  const int tile_lo = min(all_tiles, (int)blockIdx.y * per), tile_hi = min(all_tiles, tile_lo + per);

  Planes<NP> qf[KS];
  {
    const T* qp = static_cast<const T*>(a.q) + qt * a.q_row + head * a.q_head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int chunk = 2 * ks + half;
      qf[ks] = raw_planes(live && 8 * chunk < a.dim ? raw_load(qp + 8 * chunk) : raw_zero<T>());
    }
  }

  fmd_f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = zero16();
  float m = -INFINITY, l = 0.f;
  const float c = a.scale * kLog2e;

  const int lt = threadIdx.x - kw * WM * 64;  // thread among those that load this group's tiles
  // The maximum follows the scores only where one outgrows it by kSlack (in log2 units; 161 us against 166 of following
  // always, 4 x 3 000 rows, 8 heads of 64, bf16): exponentials up to 2^kSlack are
  // as exact as those below one, and the sums are rescaled a few times per row instead of once per tile.
  constexpr float kSlack = 8.f;
  const float slack = fminf(kSlack / c, 0x1p127f);  // finite for the smallest scale too: -inf + slack stays below any score

  const int lane_r = Tile::lane_rows(), lane_c = Tile::lane_cols();
  auto step = [&](auto last, const __bf16* ks_, int tile) {
    constexpr bool kLast = decltype(last)::value;  // a row may not see all of the tile
    int lr = lane_r, lc = lane_c;
    asm volatile("" : "+v"(lr), "+v"(lc));  // addresses formed here, not kept in registers
    const __bf16* vs_ = ks_ + Tile::SIZE;
    const int j0 = tile * BN;
    fmd_f32x16 s[JB];
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      s[j] = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s[j] = mma(Tile::rows(ks_, lr, 32 * j, ks), qf[ks], s[j]);
    }
    if (kLast && j0 + BN > least) {  // some row does not see all of the tile
      const int left = sees - j0 - 4 * half;
#pragma unroll
      for (int j = 0; j < JB; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (32 * j + prod_row(v, 0) >= left) s[j][v] = -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) top = fmaxf(top, s[j][v]);
    top = max_halves(top);
    if (__any(top > m + slack)) {
      top = fmaxf(top, m);
      const float fade = exp2_hw(fmaf(m, c, top == -INFINITY ? 0.f : -top * c));
      l *= fade;
      m = top;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] *= fade;
    }
    const float base = m == -INFINITY ? 0.f : m * c;  // a row that has seen nothing yet: all exponents -inf
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const float p = exp2_hw(fmaf(s[j][v], c, -base));
        s[j][v] = p;
        sum[v & 1] += p;
      }
    l += sum[0] + sum[1];  // of this lane's half of the keys
    uint32_t bad[JB] = {}, any_bad = 0;
    if (kLast && CAUSAL && j0 + BN > least) {
#pragma unroll
      for (int j = 0; j < JB; ++j) any_bad |= bad[j] = rows_not_finite<Tile>(vs_ + 32 * j * Tile::LD);
    }
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = s[j][8 * step + e];
        Planes<NP> pf, rest;
        planes_of(x, pf);
        if (kTwoParts) rest = rest_of(x, pf);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          Planes<NP> vc = Tile::cols(vs_, lc, 32 * j + 16 * step, d);
          if (kLast && CAUSAL && any_bad) vc = finite_part<NP>(vc);
          o[d] = mma(vc, pf, o[d]);
          if (kTwoParts) o[d] = mma(vc, rest, o[d]);
        }
      }
    if (kLast && CAUSAL && any_bad) {
#pragma unroll
      for (int j = 0; j < JB; ++j) mark_not_finite<Tile>(o, vs_ + 32 * j * Tile::LD, bad[j], 0, sees - j0 - 32 * j);
    }
  };

  const int rounds = (tile_hi - tile_lo + KW - 1) / KW;  // the same for every wave
  if constexpr (DMA) {
    using Dma = AttnDma<NP, BN, DP, 64 * WM>;
    uint32_t k_at[2], v_at[2];
    Dma::offsets(lt, kv.x_row, k_at);
    Dma::offsets(lt, kv.y_row, v_at);
    // the tile that is loaded next; one past the last reads nothing
    const __bf16* kp = kv.x + (sg.k0 + (int64_t)(tile_lo + kw) * BN) * kv.x_row + kvh * kv.x_head;
    const __bf16* vp = kv.y + (sg.k0 + (int64_t)(tile_lo + kw) * BN) * kv.y_row + kvh * kv.y_head;
    const int64_t k_by = (int64_t)KW * BN * kv.x_row, v_by = (int64_t)KW * BN * kv.y_row;
    auto issue = [&](int tile, __bf16* to) {
      const int n = tile < tile_hi ? sg.nk - tile * BN : 0;
      Dma::issue(kp, kv.x_row, n, a.dim, lt, k_at, to);
      Dma::issue(vp, kv.y_row, n, a.dim, lt, v_at, to + Tile::SIZE);
      kp += k_by;
      vp += v_by;
    };
    __bf16 *st0 = lds + kw * 2 * Tile::SIZE, *st1 = lds2 + kw * 2 * Tile::SIZE;
    auto round = [&](auto last, int it, const __bf16* here, __bf16* next) {
      const int tile = tile_lo + it * KW + kw;
      __builtin_amdgcn_s_waitcnt(kWaitVm0);  // this wave's part of the tile has landed
      __syncthreads();                       // everyone's has, and the other buffer is read
      if (it + 1 < rounds) issue(tile + KW, next);
      if (tile < tile_hi) step(last, here, tile);
    };
    if (rounds > 0) issue(tile_lo + kw, st0);
    int it = 0;
    if constexpr (CAUSAL)  // rounds whose tiles every row sees all of: the masks' part is left out of their code
      for (const int full = (least / BN - tile_lo) / KW; it + 2 <= full && it + 2 <= rounds; it += 2) {
        round(std::false_type(), it, st0, st1);
        round(std::false_type(), it + 1, st1, st0);
      }
    for (; it < rounds; it += 2) {
      round(std::true_type(), it, st0, st1);
      if (it + 1 < rounds) round(std::true_type(), it + 1, st1, st0);
    }
  } else {
    __bf16* st = lds + kw * 2 * Tile::SIZE;
    const T* kb = static_cast<const T*>(a.k) + sg.k0 * a.k_row + kvh * a.k_head;
    const T* vb = static_cast<const T*>(a.v) + sg.k0 * a.v_row + kvh * a.v_head;
    AttnLoad<T, NP, BN, DP, 64 * WM> kl, vl;
    auto issue = [&](int tile) {
      const int j0 = tile * BN, n = tile < tile_hi ? sg.nk - j0 : 0;
      kl.load(lt, a.dim, [&](int i) { return i < n ? kb + (int64_t)(j0 + i) * a.k_row : nullptr; });
      vl.load(lt, a.dim, [&](int i) { return i < n ? vb + (int64_t)(j0 + i) * a.v_row : nullptr; });
    };
    if (rounds > 0) issue(tile_lo + kw);
    for (int it = 0; it < rounds; ++it) {
      const int tile = tile_lo + it * KW + kw;
      __syncthreads();  // the tiles before are read
      kl.store(st, lt);
      vl.store(st + Tile::SIZE, lt);
      __syncthreads();
      if (it + 1 < rounds) issue(tile + KW);
      if (tile < tile_hi) step(std::true_type(), st, tile);
    }
  }
  l = add_halves(l);

  if constexpr (KW > 1) {  // join the key groups, in their order
    float* mg = reinterpret_cast<float*>(lds);
    __syncthreads();
    if (kw > 0) {
      float* w = mg + ((kw - 1) * WM + wm) * (DB * 16 + 2) * 64 + lane;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) w[(d * 16 + v) * 64] = o[d][v];
      w[DB * 16 * 64] = m;
      w[(DB * 16 + 1) * 64] = l;
    }
    __syncthreads();
    if (kw > 0) return;
#pragma unroll
    for (int g = 0; g < KW - 1; ++g) {
      const float* w = mg + (g * WM + wm) * (DB * 16 + 2) * 64 + lane;
      const float gm = w[DB * 16 * 64], gl = w[(DB * 16 + 1) * 64];
      const float top = fmaxf(m, gm), base = top == -INFINITY ? 0.f : top * c;
      const float fa = exp2_hw(fmaf(m, c, -base)), fb = exp2_hw(fmaf(gm, c, -base));
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] = o[d][v] * fa + w[(d * 16 + v) * 64] * fb;
      l = l * fa + gl * fb;
      m = top;
    }
  }
  if (!live) return;

  if (splits == 1) {
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // a row that sees no key gives zero
    const int64_t at = (qt * a.heads + head) * a.dim;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int col = 32 * d + 8 * r + 4 * half;
        if (col >= a.dim) continue;
        const float x[4] = {o[d][4 * r] * inv, o[d][4 * r + 1] * inv, o[d][4 * r + 2] * inv, o[d][4 * r + 3] * inv};
        store4<T>(out + at + col, x[0], x[1], x[2], x[3]);
        saved_residual<T>(saved, at + col, x);
      }
    if (saved.base && half == 0) {
      saved.base[head * a.tq + qt] = m == -INFINITY ? 0.f : m * c;
      saved.inverse[head * a.tq + qt] = inv;
    }
  } else {
    const int64_t at = ((int64_t)blockIdx.y * a.tq + qt) * a.heads + head;
    float* op = part_o + at * a.dim;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int col = 32 * d + 8 * r + 4 * half;
        if (col < a.dim) store4<float>(op + col, o[d][4 * r], o[d][4 * r + 1], o[d][4 * r + 2], o[d][4 * r + 3]);
      }
    if (half == 0) {
      part_m[at] = m;
      part_l[at] = l;
    }
  }
}

// The splits of a row joined in their order: one wave per (query, head). The lanes hold the splits' maxima and sums (at most 64
// splits), then columns; the loads of eight splits are in flight together. Latency bounds it: 4.4 us for 4 splits of 256 rows of
// 128.
constexpr int kMaxSplits = 64;

template <typename T>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a, int splits, const float* part_o, const float* part_m,
                                                        const float* part_l, T* out, AttnSaved saved) {
  const int64_t n = a.tq * a.heads, at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (at >= n) return;
  const float c = a.scale * kLog2e;
  const float m = lane < splits ? part_m[lane * n + at] : -INFINITY, pl = lane < splits ? part_l[lane * n + at] : 0.f;
  const float top = wave_max(m), base = top == -INFINITY ? 0.f : top * c;
  const float f = exp2_hw(fmaf(m, c, -base));
  const float l = wave_sum(f * pl);
  float o[2] = {0.f, 0.f};
  for (int s0 = 0; s0 < splits; s0 += 8) {
    float x[8][2];
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int col = lane + 64 * k;
        x[s][k] = s0 + s < splits && col < a.dim ? part_o[((s0 + s) * n + at) * a.dim + col] : 0.f;
      }
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const float fs = __shfl(f, (s0 + s) & 63, 64);
#pragma unroll
      for (int k = 0; k < 2; ++k) o[k] += fs * x[s][k];
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (lane + 64 * k < a.dim) {
      const int64_t i = at * a.dim + lane + 64 * k;
      const float x = o[k] * inv;
      out[i] = (T)x;
      if (sizeof(T) == 2 && saved.residual) static_cast<T*>(saved.residual)[i] = (T)(x - (float)(T)x);
    }
  if (saved.base && lane == 0) {
    saved.base[(at % a.heads) * a.tq + at / a.heads] = base;
    saved.inverse[(at % a.heads) * a.tq + at / a.heads] = inv;
  }
}

// ------------------------------------------------------------------------------------ backward

// Per query and head: delta = g . o, and the offset that the exponents are formed with: base - log2(inverse) for bf16 (the
// rounding of the sum, 2^-24 of it, is far below the rounding of P), base for fp32, which multiplies by the inverse; +inf for
// a row that sees nothing. 16 lanes a row. Memory bounds it: 8 192 rows of 16 heads of 128, bf16, 21 us (100 MB).
template <typename T>
__global__ void __launch_bounds__(256) attn_delta_kernel(AttnBwd b, int64_t tq, int heads, int dim, int64_t block0, float* rows) {
  const int64_t at = (block0 + blockIdx.x) * 16 + (threadIdx.x >> 4);
  const int sub = threadIdx.x & 15;
  const int64_t tok = at / heads;
  const int head = (int)(at % heads);
  float s = 0.f;
  if (tok < tq) {
    const T *gp = static_cast<const T*>(b.g) + tok * b.g_row + head * b.g_head, *op = static_cast<const T*>(b.out) + at * dim;
    const T* rp = static_cast<const T*>(b.saved.residual) + at * dim;
    const int d = sub * 8;
    if (d < dim) {
      const Raw8<T> x = raw_load(gp + d), y = raw_load(op + d), z = sizeof(T) == 2 ? raw_load(rp + d) : raw_zero<T>();
      const T *xe = reinterpret_cast<const T*>(&x), *ye = reinterpret_cast<const T*>(&y), *ze = reinterpret_cast<const T*>(&z);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += (float)xe[e] * ((float)ye[e] + (float)ze[e]);
    }
  }
  s = lanes_sum<16>(s);
  if (tok < tq && sub == 0) {
    const int64_t i = head * tq + tok;
    const float inv = b.saved.inverse[i];
    rows[i] = inv == 0.f ? INFINITY : b.saved.base[i] - (sizeof(T) == 2 ? __log2f(inv) : 0.f);
    rows[heads * tq + i] = s;
  }
}

// Gradients of keys and values. One workgroup: 32 WM keys of one key head; wave (wm, rw) holds 32 keys and walks the
// tiles rw, rw + RW, ... of 32 queries, of one query head of the group after the other. S = Q K^T (lane: a key, registers:
// query rows), so exp(S - lse) and dS are the operands of gv^T = G^T P and gk^T = Q^T dS, whose sums run over all query heads of
// the group. For bf16, P and dS are operands in two bf16 parts; sums are fp32.
// Measured: bf16, causal, 4 sequences of 8 192 rows together, 16 heads on 4 of 128: 280 us, 525 TFLOP/s of the 8 D operations, 790
// with the second parts', matrix pipes busy 47 % of the time: two waves a SIMD, for which the two sums take half of the
// registers, wait on each other's rounds. fp32, 5 systems of 5 000 rows, 4 heads of 64: 150 us, 150 TFLOP/s. Two waves of keys
// and four of rows in one workgroup, so that a tile's copy serves both and each SIMD has two waves.
template <typename T, int DP, int WM, int RW, bool DMA, bool CAUSAL>
__global__ void __launch_bounds__(64 * WM * RW, AttnType<T>::planes == 1 ? 2 : attn_waves(AttnType<T>::planes, DP, 2)) attn_bwd_kv_kernel(AttnArgs a, AttnBwd b, AttnTiles qg,
                                                                                              int splits, float* part, T* gk, T* gv) {
  constexpr int NP = AttnType<T>::planes, DB = DP / 32, KS = DP / 16, BR = 32;
  constexpr bool kTwoParts = NP == 1;
  using Tile = AttnTile<NP, BR, DP>;
  constexpr int kStats = NP == 3 ? 4 * BR : 2 * BR;  // offset, delta (inverse and nothing) of BR rows
  constexpr int kGroup = 2 * Tile::SIZE + 2 * kStats;  // in bf16 units
  constexpr int MB = DB < 2 ? DB : 2;  // column blocks of a gradient that are joined at a time
  constexpr int kMerge = (RW - 1) * WM * MB * 16 * 64 * 2;
  __shared__ __attribute__((aligned(16))) __bf16 lds[RW * kGroup > kMerge ? RW * kGroup : kMerge];
  __shared__ __attribute__((aligned(16))) __bf16 lds2[DMA ? RW * kGroup : 8];
  // the values of the workgroup's keys stay in LDS where they and the keys do not both fit into registers (beside the masks of a
  // causal call, from 96 columns on)
  constexpr bool kLdsV = NP == 1 && DP > (CAUSAL ? 64 : 96) && RW > 1;
  using VTile = AttnTile<NP, 32 * WM, DP>;
  __shared__ __attribute__((aligned(16))) __bf16 lds_v[kLdsV ? VTile::SIZE : 8];

  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, rw = wave / WM;
  const uint32_t block = a.block0 + blockIdx.x;
  const int kvh = block % a.kv_heads;
  int64_t first;
  const int ext = attn_find(a.k_off, a.segments, a.tk, 1, 32 * WM, block / a.kv_heads, &first, WaveLanes());
  AttnSegment sg = attn_segment(a, ext);
  if (!attn_real(a, ext)) sg.nq = 0;
  if (first >= sg.nk) return;
  const int key0 = (int)first, key = key0 + 32 * wm + (lane & 31);
  const bool live = key < sg.nk;
  const int64_t kt = sg.k0 + (live ? key : 0);
  const int shift = sg.nk - sg.nq;
  // the first query that sees this key and the first that sees all keys of the workgroup; the tiles of a head that see any
  const int from = CAUSAL ? max(0, key - shift) : 0;
  const int full = CAUSAL ? max(0, key0 + 32 * WM - 1 - shift) : 0;
  const int tile_lo = CAUSAL ? min(sg.nq, max(0, key0 - shift)) / BR : 0;
  const int head_tiles = (sg.nq + BR - 1) / BR - tile_lo;
  // this split's part of the tiles of all heads
  const int per = (head_tiles * a.group + splits - 1) / splits, first_tile = blockIdx.y * per;
  const int all_tiles = min(head_tiles * a.group, first_tile + per);

  Planes<NP> kf[KS], vf[kLdsV ? 1 : KS];
  {
    const T* kp = static_cast<const T*>(a.k) + kt * a.k_row + kvh * a.k_head;
    const T* vp = static_cast<const T*>(a.v) + kt * a.v_row + kvh * a.v_head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int chunk = 2 * ks + half;
      const bool ok = live && 8 * chunk < a.dim;
      kf[ks] = raw_planes(ok ? raw_load(kp + 8 * chunk) : raw_zero<T>());
      const Planes<NP> v = raw_planes(ok ? raw_load(vp + 8 * chunk) : raw_zero<T>());
      if constexpr (kLdsV) {
        if (rw == 0) VTile::put(lds_v, 32 * wm + (lane & 31), chunk, v);  // read after the first barrier
      } else {
        vf[ks] = v;
      }
    }
  }
  fmd_f32x16 ak[DB], av[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) ak[d] = av[d] = zero16();
  const float c = a.scale * kLog2e;

  const int lt = threadIdx.x - rw * WM * 64;
  // the tile that is loaded next: its number, first query, and where its rows and their statistics lie
  using S = std::conditional_t<DMA, __bf16, T>;
  const int64_t q_ld = DMA ? qg.x_row : a.q_row, g_ld = DMA ? qg.y_row : b.g_row;
  const int64_t q_hd = DMA ? qg.x_head : a.q_head, g_hd = DMA ? qg.y_head : b.g_head;
  int next_tile = first_tile + rw, next_row = (tile_lo + next_tile) * BR;
  const S* qp = static_cast<const S*>(DMA ? qg.x : a.q) + (sg.q0 + next_row) * q_ld + (int64_t)kvh * a.group * q_hd;
  const S* gp = static_cast<const S*>(DMA ? qg.y : b.g) + (sg.q0 + next_row) * g_ld + (int64_t)kvh * a.group * g_hd;
  int64_t stat_at = (int64_t)kvh * a.group * a.tq + sg.q0 + next_row;
  const float *offset = b.rows, *delta = b.rows + a.heads * a.tq;
  const int64_t q_by = (int64_t)RW * BR * q_ld, g_by = (int64_t)RW * BR * g_ld;
  const int64_t q_head = q_hd - (int64_t)head_tiles * BR * q_ld, g_head = g_hd - (int64_t)head_tiles * BR * g_ld;
  auto wrap = [&] {
    while (next_row >= (tile_lo + head_tiles) * BR && next_tile < all_tiles) {  // the next head's tiles
      next_row -= head_tiles * BR;
      qp += q_head;
      gp += g_head;
      stat_at += a.tq - head_tiles * BR;
    }
  };
  auto advance = [&] {
    next_tile += RW;
    next_row += RW * BR;
    qp += q_by;
    gp += g_by;
    stat_at += RW * BR;
    wrap();
  };
  const int lane_r = Tile::lane_rows(), lane_c = Tile::lane_cols();
  auto step = [&](auto partial, const __bf16* qs, int r0) {
    constexpr bool kPartial = decltype(partial)::value;  // some key of the workgroup may not be seen by some row
    int lr = lane_r, lc = lane_c;
    if constexpr (kLdsV) asm volatile("" : "+v"(lr), "+v"(lc));  // addresses formed here, not kept in registers
    const __bf16* gs = qs + Tile::SIZE;
    const float* stat = reinterpret_cast<const float*>(gs + Tile::SIZE);
    fmd_f32x16 s = zero16(), dp = zero16();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = mma(Tile::rows(qs, lr, 0, ks), kf[ks], s);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      dp = mma(Tile::rows(gs, lr, 0, ks), kLdsV ? VTile::rows(lds_v, lr, 32 * wm, ks) : vf[kLdsV ? 0 : ks], dp);
    uint32_t bad = 0;
    if (kPartial && r0 < full && not_finite(s, dp)) bad = rows_not_finite<Tile>(qs) | rows_not_finite<Tile>(gs);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float4 ls = *reinterpret_cast<const float4*>(stat + 8 * r + 4 * half);
      const float4 dl = *reinterpret_cast<const float4*>(stat + BR + 8 * r + 4 * half);
      const float4 iv = NP == 3 ? *reinterpret_cast<const float4*>(stat + 2 * BR + 8 * r + 4 * half) : make_float4(1.f, 1.f, 1.f, 1.f);
      const float le[4] = {ls.x, ls.y, ls.z, ls.w}, de[4] = {dl.x, dl.y, dl.z, dl.w}, ie[4] = {iv.x, iv.y, iv.z, iv.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = 4 * r + e;
        float p = exp2_hw(fmaf(s[v], c, -le[e]));
        if (NP == 3) p *= ie[e];
        s[v] = p;
        dp[v] = p * (dp[v] - de[e]);
      }
    }
    if (kPartial && r0 < full) {
      const int hidden = from - r0 - 4 * half;
#pragma unroll
      for (int v = 0; v < 16; ++v)
        if (prod_row(v, 0) < hidden) s[v] = dp[v] = 0.f;
    }
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      float x[8], y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = s[8 * step + e];
        y[e] = dp[8 * step + e];
      }
      Planes<NP> pf, df, pf_rest, df_rest;
      planes_of(x, pf);
      planes_of(y, df);
      if (kTwoParts) pf_rest = rest_of(x, pf), df_rest = rest_of(y, df);
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        Planes<NP> gc = Tile::cols(gs, lc, 16 * step, d);
        if (kPartial && bad) gc = finite_part<NP>(gc);
        av[d] = mma(gc, pf, av[d]);
        if (kTwoParts) av[d] = mma(gc, pf_rest, av[d]);
        Planes<NP> qc = Tile::cols(qs, lc, 16 * step, d);
        if (kPartial && bad) qc = finite_part<NP>(qc);
        ak[d] = mma(qc, df, ak[d]);
        if (kTwoParts) ak[d] = mma(qc, df_rest, ak[d]);
      }
    }
    if (kPartial && bad) {
      mark_not_finite<Tile>(av, gs, bad, from - r0, BR);
      mark_not_finite<Tile>(ak, qs, bad, from - r0, BR);
    }
  };

  const int rounds = (max(0, all_tiles - first_tile) + RW - 1) / RW;
  wrap();
  if constexpr (DMA) {
    using Dma = AttnDma<NP, BR, DP, 64 * WM>;
    static_assert(NP == 1 || WM > 1, "the second wave copies the inverses");
    __bf16 *st0 = lds + rw * kGroup, *st1 = lds2 + rw * kGroup;
    uint32_t q_off[2], g_off[2];
    Dma::offsets(lt, q_ld, q_off);
    Dma::offsets(lt, g_ld, g_off);
    auto issue = [&](__bf16* to) {
      const int n = next_tile < all_tiles ? sg.nq - next_row : 0;
      Dma::issue(qp, q_ld, n, a.dim, lt, q_off, to);
      Dma::issue(gp, g_ld, n, a.dim, lt, g_off, to + Tile::SIZE);
      if (wm == 0 || (NP == 3 && wm == 1)) {  // offsets and deltas (inverses): lane i of each half the row i
        int i = lane;
        asm volatile("" : "+v"(i));
        const bool second = i >= 32;
        i &= 31;
        const float* p = (wm == 1 ? b.saved.inverse : second ? delta : offset) + stat_at + i;
        if (i >= n) p = g_attn_no_row + (second || wm == 1);
        asm volatile("" : "+v"(p));
        Dma::copy4(p, to + 2 * Tile::SIZE + (wm == 1 ? 4 * BR : 0));
      }
    };
    auto round = [&](auto partial, int it, const __bf16* here, __bf16* next) {
      const int tile = next_tile, r0 = next_row;
      __builtin_amdgcn_s_waitcnt(kWaitVm0);
      __syncthreads();
      advance();
      if (it + 1 < rounds) issue(next);
      if (tile < all_tiles) step(partial, here, r0);
    };
    if (rounds > 0) issue(st0);
    if constexpr (CAUSAL) {
      // every head's tiles begin with those that some key is not seen by; the masks' part is left out of the others' code
      const int hidden_tiles = (full + BR - 1) / BR - tile_lo;
      int at = head_tiles > 0 ? first_tile % head_tiles : 0;
      for (int it = 0; it < rounds;) {
        for (; it < rounds && (at < hidden_tiles || at + 2 * RW > head_tiles); it += 2) {
          round(std::true_type(), it, st0, st1);
          if (it + 1 < rounds) round(std::true_type(), it + 1, st1, st0);
          for (at += 2 * RW; at >= head_tiles;) at -= head_tiles;
        }
        for (; it < rounds && at >= hidden_tiles && at + 2 * RW <= head_tiles; it += 2, at += 2 * RW) {
          round(std::false_type(), it, st0, st1);
          if (it + 1 < rounds) round(std::false_type(), it + 1, st1, st0);
        }
        if (at >= head_tiles) at = 0;
      }
    } else {
      for (int it = 0; it < rounds; it += 2) {
        round(std::false_type(), it, st0, st1);
        if (it + 1 < rounds) round(std::false_type(), it + 1, st1, st0);
      }
    }
  } else {
    __bf16* qs = lds + rw * kGroup;
    AttnLoad<T, NP, BR, DP, 64 * WM> ql, gl;
    constexpr int kStatLoads = (kStats + 64 * WM - 1) / (64 * WM);
    float st[kStatLoads];
    auto issue = [&] {
      const int n = next_tile < all_tiles ? sg.nq - next_row : 0;
      ql.load(lt, a.dim, [&](int i) { return i < n ? qp + i * q_ld : nullptr; });
      gl.load(lt, a.dim, [&](int i) { return i < n ? gp + i * g_ld : nullptr; });
#pragma unroll
      for (int k = 0; k < kStatLoads; ++k) {
        const int x = lt + k * 64 * WM, i = x % BR, which = x / BR;
        const float* p = which == 0 ? offset : which == 1 ? delta : b.saved.inverse;
        st[k] = which < 3 && i < n ? p[stat_at + i] : which == 0 ? INFINITY : 0.f;
      }
    };
    if (rounds > 0) issue();
    for (int it = 0; it < rounds; ++it) {
      const int tile = next_tile, r0 = next_row;
      __syncthreads();
      ql.store(qs, lt);
      gl.store(qs + Tile::SIZE, lt);
#pragma unroll
      for (int k = 0; k < kStatLoads; ++k)
        if (lt + k * 64 * WM < kStats) reinterpret_cast<float*>(qs + 2 * Tile::SIZE)[lt + k * 64 * WM] = st[k];
      __syncthreads();
      advance();
      if (it + 1 < rounds) issue();
      if (tile < all_tiles) step(std::bool_constant<CAUSAL>(), qs, r0);
    }
  }

  if constexpr (RW > 1) {  // add the row groups, in their order
    float* mg = reinterpret_cast<float*>(lds);
    auto join = [&](fmd_f32x16(&acc)[DB]) {
#pragma unroll
      for (int d0 = 0; d0 < DB; d0 += MB) {
        __syncthreads();
        float* mine = mg + ((rw - 1) * WM + wm) * MB * 16 * 64 + lane;
        if (rw > 0) {
#pragma unroll
          for (int d = d0; d < d0 + MB && d < DB; ++d)
#pragma unroll
            for (int v = 0; v < 16; ++v) mine[((d - d0) * 16 + v) * 64] = acc[d][v];
        }
        __syncthreads();
        if (rw == 0) {
#pragma unroll
          for (int g = 0; g < RW - 1; ++g) {
            const float* w = mg + (g * WM + wm) * MB * 16 * 64 + lane;
#pragma unroll
            for (int d = d0; d < d0 + MB && d < DB; ++d)
#pragma unroll
              for (int v = 0; v < 16; ++v) acc[d][v] += w[((d - d0) * 16 + v) * 64];
          }
        }
      }
    };
    join(ak);
    join(av);
    if (rw > 0) return;
  }
  if (!live) return;
  const int64_t at = (kt * a.kv_heads + kvh) * a.dim, all = a.tk * a.kv_heads * a.dim;
  float* pk = part + (int64_t)blockIdx.y * 2 * all + at;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int col = 32 * d + 8 * r + 4 * half;
      if (col >= a.dim) continue;
      const float f = a.scale;
      if (splits > 1) {
        store4<float>(pk + col, ak[d][4 * r] * f, ak[d][4 * r + 1] * f, ak[d][4 * r + 2] * f, ak[d][4 * r + 3] * f);
        store4<float>(pk + all + col, av[d][4 * r], av[d][4 * r + 1], av[d][4 * r + 2], av[d][4 * r + 3]);
        continue;
      }
      store4<T>(gk + at + col, ak[d][4 * r] * f, ak[d][4 * r + 1] * f, ak[d][4 * r + 2] * f, ak[d][4 * r + 3] * f);
      store4<T>(gv + at + col, av[d][4 * r], av[d][4 * r + 1], av[d][4 * r + 2], av[d][4 * r + 3]);
    }
}

// Gradient of the queries: the forward's walk with S^T = K Q^T and dP^T = V G^T, then gq^T = K^T dS^T (dS in two parts for
// bf16). Measured in the cases above: bf16 160 us, 690 TFLOP/s of the 6 D operations, 920 with the second part's, matrix pipes busy 54 %
// of the time; fp32 113 us, 149 TFLOP/s.
template <typename T, int DP, int WM, int KW, bool DMA, bool CAUSAL>
__global__ void __launch_bounds__(64 * WM * KW, attn_waves(AttnType<T>::planes, DP, 1)) attn_bwd_q_kernel(AttnArgs a, AttnBwd b, AttnTiles kv,
                                                                                             int64_t tiles, int splits, float* part, T* gq) {
  constexpr int NP = AttnType<T>::planes, DB = DP / 32, KS = DP / 16, BN = WM > 1 && NP == 1 ? 64 : 32;
  constexpr bool kTwoParts = NP == 1;
  using Tile = AttnTile<NP, BN, DP>;
  constexpr int kTiles = 2 * KW * Tile::SIZE, kMerge = (KW - 1) * WM * 16 * 64 * 2;
  __shared__ __attribute__((aligned(16))) __bf16 lds[kTiles > kMerge ? kTiles : kMerge];
  __shared__ __attribute__((aligned(16))) __bf16 lds2[DMA ? kTiles : 8];

  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, kw = wave / WM;
  const uint32_t block = a.block0 + blockIdx.x;
  const int kvh = block % a.kv_heads;
  int64_t t = block / a.kv_heads;
  if (CAUSAL) t = tiles - 1 - t;
  int64_t first;
  const int ext = attn_find(a.q_off, a.segments, a.tq, a.group, 32 * WM, t, &first, WaveLanes());
  AttnSegment sg = attn_segment(a, ext);
  if (!attn_real(a, ext)) sg.nk = 0;
  const int rows = sg.nq * a.group;
  if (first >= rows) return;
  const int row0 = (int)first, row = row0 + 32 * wm + (lane & 31);
  const bool live = row < rows;
  const int tok = attn_token(a, live ? row : rows - 1), head = kvh * a.group + (live ? row : rows - 1) - tok * a.group;
  const int64_t qt = sg.q0 + tok;
  const int shift = sg.nk - sg.nq;
  const int sees = CAUSAL ? max(0, min(sg.nk, tok + shift + 1)) : sg.nk;
  const int last_row = min(row0 + 32 * WM, rows) - 1;
  const int reach = CAUSAL ? max(0, min(sg.nk, attn_token(a, last_row) + shift + 1)) : sg.nk;
  const int least = CAUSAL ? max(0, min(sg.nk, attn_token(a, row0) + shift + 1)) : sg.nk;
  const int per = ((reach + BN - 1) / BN + splits - 1) / splits;
  const int tile_lo = blockIdx.y * per, tile_hi = min((reach + BN - 1) / BN, tile_lo + per);

  Planes<NP> qf[KS], gf[KS];
  {
    const T* qp = static_cast<const T*>(a.q) + qt * a.q_row + head * a.q_head;
    const T* gp = static_cast<const T*>(b.g) + qt * b.g_row + head * b.g_head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int chunk = 2 * ks + half;
      const bool ok = live && 8 * chunk < a.dim;
      qf[ks] = raw_planes(ok ? raw_load(qp + 8 * chunk) : raw_zero<T>());
      gf[ks] = raw_planes(ok ? raw_load(gp + 8 * chunk) : raw_zero<T>());
    }
  }
  // fp32: P = exp2(s - offset) inverse, the inverse taken into the other factor of dS
  const float inv = NP == 3 ? b.saved.inverse[head * a.tq + qt] : 1.f, ls = b.rows[head * a.tq + qt];
  const float dl = b.rows[(a.heads + head) * a.tq + qt] * inv;
  fmd_f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = zero16();
  const float c = a.scale * kLog2e;

  const int lt = threadIdx.x - kw * WM * 64;
  const int lane_r = Tile::lane_rows(), lane_c = Tile::lane_cols();
  auto step = [&](auto last, const __bf16* ks_, int tile) {
    constexpr bool kLast = decltype(last)::value;  // a row may not see all of the tile
    int lr = lane_r, lc = lane_c;
    asm volatile("" : "+v"(lr), "+v"(lc));  // addresses formed here, not kept in registers
    const __bf16* vs_ = ks_ + Tile::SIZE;
#pragma unroll
    for (int jb = 0; jb < BN; jb += 32) {
      const int j0 = tile * BN + jb;
      fmd_f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = mma(Tile::rows(ks_, lr, jb, ks), qf[ks], s);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) dp = mma(Tile::rows(vs_, lr, jb, ks), gf[ks], dp);
#pragma unroll
      for (int v = 0; v < 16; ++v) s[v] = exp2_hw(fmaf(s[v], c, -ls)) * (NP == 3 ? fmaf(dp[v], inv, -dl) : dp[v] - dl);
      uint32_t bad = 0;
      if (kLast && j0 + 32 > least) {
        const int left = sees - j0 - 4 * half;
        if (CAUSAL) bad = rows_not_finite<Tile>(ks_ + jb * Tile::LD);
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (prod_row(v, 0) >= left) s[v] = 0.f;
      }
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = s[8 * step + e];
        Planes<NP> df, rest;
        planes_of(y, df);
        if (kTwoParts) rest = rest_of(y, df);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          Planes<NP> kc = Tile::cols(ks_, lc, jb + 16 * step, d);
          if (kLast && CAUSAL && bad) kc = finite_part<NP>(kc);
          o[d] = mma(kc, df, o[d]);
          if (kTwoParts) o[d] = mma(kc, rest, o[d]);
        }
      }
      if (kLast && CAUSAL && bad) mark_not_finite<Tile>(o, ks_ + jb * Tile::LD, bad, 0, sees - j0);
    }
  };
  const int rounds = (max(0, tile_hi - tile_lo) + KW - 1) / KW;
  if constexpr (DMA) {
    using Dma = AttnDma<NP, BN, DP, 64 * WM>;
    __bf16 *st0 = lds + kw * 2 * Tile::SIZE, *st1 = lds2 + kw * 2 * Tile::SIZE;
    uint32_t k_at[2], v_at[2];
    Dma::offsets(lt, kv.x_row, k_at);
    Dma::offsets(lt, kv.y_row, v_at);
    const __bf16* kp = kv.x + (sg.k0 + (int64_t)(tile_lo + kw) * BN) * kv.x_row + kvh * kv.x_head;
    const __bf16* vp = kv.y + (sg.k0 + (int64_t)(tile_lo + kw) * BN) * kv.y_row + kvh * kv.y_head;
    const int64_t k_by = (int64_t)KW * BN * kv.x_row, v_by = (int64_t)KW * BN * kv.y_row;
    auto issue = [&](int tile, __bf16* to) {
      const int n = tile < tile_hi ? sg.nk - tile * BN : 0;
      Dma::issue(kp, kv.x_row, n, a.dim, lt, k_at, to);
      Dma::issue(vp, kv.y_row, n, a.dim, lt, v_at, to + Tile::SIZE);
      kp += k_by;
      vp += v_by;
    };
    auto round = [&](auto last, int it, const __bf16* here, __bf16* next) {
      const int tile = tile_lo + it * KW + kw;
      __builtin_amdgcn_s_waitcnt(kWaitVm0);
      __syncthreads();
      if (it + 1 < rounds) issue(tile + KW, next);
      if (tile < tile_hi) step(last, here, tile);
    };
    if (rounds > 0) issue(tile_lo + kw, st0);
    int it = 0;
    if constexpr (CAUSAL)  // rounds whose tiles every row sees all of: the masks' part is left out of their code
      for (const int full = (least / BN - tile_lo) / KW; it + 2 <= full && it + 2 <= rounds; it += 2) {
        round(std::false_type(), it, st0, st1);
        round(std::false_type(), it + 1, st1, st0);
      }
    for (; it < rounds; it += 2) {
      round(std::true_type(), it, st0, st1);
      if (it + 1 < rounds) round(std::true_type(), it + 1, st1, st0);
    }
  } else {
    __bf16* st = lds + kw * 2 * Tile::SIZE;
    const T* kb = static_cast<const T*>(a.k) + sg.k0 * a.k_row + kvh * a.k_head;
    const T* vb = static_cast<const T*>(a.v) + sg.k0 * a.v_row + kvh * a.v_head;
    AttnLoad<T, NP, BN, DP, 64 * WM> kl, vl;
    auto issue = [&](int tile) {
      const int j0 = tile * BN, n = tile < tile_hi ? sg.nk - j0 : 0;
      kl.load(lt, a.dim, [&](int i) { return i < n ? kb + (int64_t)(j0 + i) * a.k_row : nullptr; });
      vl.load(lt, a.dim, [&](int i) { return i < n ? vb + (int64_t)(j0 + i) * a.v_row : nullptr; });
    };
    if (rounds > 0) issue(tile_lo + kw);
    for (int it = 0; it < rounds; ++it) {
      const int tile = tile_lo + it * KW + kw;
      __syncthreads();
      kl.store(st, lt);
      vl.store(st + Tile::SIZE, lt);
      __syncthreads();
      if (it + 1 < rounds) issue(tile + KW);
      if (tile < tile_hi) step(std::true_type(), st, tile);
    }
  }
  if constexpr (KW > 1) {  // add the key groups, in their order, a column block at a time
    float* mg = reinterpret_cast<float*>(lds) + lane;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      __syncthreads();
      if (kw > 0) {
#pragma unroll
        for (int v = 0; v < 16; ++v) mg[(((kw - 1) * WM + wm) * 16 + v) * 64] = o[d][v];
      }
      __syncthreads();
      if (kw == 0) {
#pragma unroll
        for (int g = 0; g < KW - 1; ++g)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[d][v] += mg[((g * WM + wm) * 16 + v) * 64];
      }
    }
    if (kw > 0) return;
  }
  if (!live) return;
  const int64_t at = (qt * a.heads + head) * a.dim;
  float* pq = part + (int64_t)blockIdx.y * a.tq * a.heads * a.dim + at;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int col = 32 * d + 8 * r + 4 * half;
      const float f = a.scale;
      if (col >= a.dim) continue;
      if (splits > 1) store4<float>(pq + col, o[d][4 * r] * f, o[d][4 * r + 1] * f, o[d][4 * r + 2] * f, o[d][4 * r + 3] * f);
      else store4<T>(gq + at + col, o[d][4 * r] * f, o[d][4 * r + 1] * f, o[d][4 * r + 2] * f, o[d][4 * r + 3] * f);
    }
}

// The splits' sums added in their order (a few us, latency), four values a thread: of x, and of y behind it in every split (or null)
template <typename T>
__global__ void __launch_bounds__(256) attn_add_kernel(const float* part, int64_t n, int splits, T* x, T* y) {
  const int64_t all = y ? 2 * n : n, i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= all) return;
  float4 s = *reinterpret_cast<const float4*>(part + i);
  for (int k = 1; k < splits; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(part + k * all + i);
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  store4<T>(i < n ? x + i : y + i - n, s.x, s.y, s.z, s.w);
}

// fp32 rows [rows, heads, dim] as planes [rows, heads, 3, dim], a thread per eight values: split once here, where the wide and
// middle tiles would split each tile in every workgroup that reads it (5 systems of 5 000 rows, 4 heads of 64: forward 160 us
// without planes, 98 with them). Memory bounds it: 16 875 rows of 4 heads of 32, two arrays, 8-10 us.
__global__ void __launch_bounds__(256) attn_split_kernel(const float* x, int64_t x_row, int64_t x_head, const float* y, int64_t y_row,
                                                         int64_t y_head, int64_t rows, int heads, int dim, __bf16* xp, __bf16* yp) {
  const int chunks = dim / 8;
  const int64_t n = rows * heads * chunks, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t rh = i / chunks, row = rh / heads;
  const int chunk = (int)(i % chunks) * 8, head = (int)(rh % heads);
  const float* src[2] = {x + row * x_row + head * x_head, y + row * y_row + head * y_head};
  __bf16* dst[2] = {xp, yp};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const Planes<3> v = raw_planes(raw_load(src[k] + chunk));
#pragma unroll
    for (int p = 0; p < 3; ++p) *reinterpret_cast<fmd_bf16x8*>(dst[k] + (rh * 3 + p) * dim + chunk) = v.p[p];
  }
}

// ------------------------------------------------------------------------------------ launches

// tiles of `bm` rows: the numbers that attn_find hands out
int64_t tile_count(int64_t rows, int group, int segments, int bm) { return rows * group / bm + segments + 2; }

// How a workgroup's waves share a tile. kWide: four waves of 32 rows each over the same keys. kNarrow: the waves take the same
// 32 rows and share the keys, for calls with too few tiles to fill the card otherwise and segments not much longer than a
// tile. kMid: two and two, fp32 only, whose narrow form splits every tile into planes in the wave that reads it (fp32 heads
// above 64 have room in LDS for wide tiles alone, and two narrow waves).
// Measured, us of forward + both halves of the VJP:
//   one segment, bf16, 8 heads of 64: 2 000 rows narrow 101, wide 148; 4 000 rows 307, 308; 8 000 rows 1 110, 976
//   ", 8 heads of 128: 1 000 rows 83, 123; 2 000 rows 242, 212; 4 000 rows 853, 475
//   ", fp32, 4 heads of 32: 2 000 rows narrow 122, mid 135, wide 142; 4 000 rows 325, 300, 436; 8 000 rows 1 157, 913, 1 063
//   ", 4 heads of 64: 1 000 rows 99, 125, 185; 2 000 rows 198, 178, 196; 8 000 rows 2 753, 1 734, 1 619
//   ", 4 heads of 128: 1 000 rows narrow 320, wide 304; 2 000 rows 805, 296
//   64 segments, 4 heads of 32, fp32: 80 rows narrow 54, mid 82, wide 67; 160 rows 102, 118, 105; 320 rows 210, 215, 193;
//   bf16: 80 rows 53, -, 54; 160 rows 57, -, 63; 320 rows 100, -, 104; 40 segments, 4 heads of 64, 200 rows 77, -, 70; 400 rows 155, -, 133
enum AttnShape { kNarrow, kMid, kWide };

AttnShape shape_of(bool f32, int dim, int64_t rows, int heads, int segments) {
  const int64_t blocks = rows / 32 * heads;
  if (rows < (int64_t)(f32 && dim <= 64 ? 192 : 64) * segments) return kNarrow;
  if (blocks >= (dim <= 64 ? (f32 ? 1024 : 900) : f32 ? 192 : 384)) return kWide;
  return f32 && dim <= 64 && blocks >= (dim <= 32 ? 384 : 224) ? kMid : kNarrow;
}

constexpr int shape_rows(AttnShape s) { return s == kWide ? 128 : s == kMid ? 64 : 32; }

// About one query per segment, and enough segments to fill the card with a wave each or so few keys that a tile is mostly
// empty: the row kernels. The more segments, the longer a wave may take over one. Measured, us of forward + VJP on the row
// kernels (tiles):
//   4 heads of 32, fp32: 10 000 segments of 18 keys 103 (1 004), 256 of 128 39 (61), 256 of 400 114 (100), 2 000 of 400 504 (762),
//   1 024 of 500 338 (455); bf16: 54 (456), 42 (49), 115 (113), 269 (845), 224 (520)
//   8 heads of 128, fp32: 153 segments of 21 keys 47 (240), of 64 104 (223), of 128 202 (404); bf16 47 (150), 113 (216), 212 (236);
//   8 heads of 32, 40 of 21 44 (48)
// These are of groups whose heads a wave takes together (1, 2 and 4; of 4: fp32, 256 segments of 128 keys, 4 heads on one of 64, 35 (95);
// bf16, 1 024 of 500, 16 heads on 4 of 128, 1 284 (2 412)). Of other groups it walks the keys for each head, and many segments of few keys
// are left to it: 8 heads on one of 64, fp32: 10 000 segments of 18 keys 285 (1 530), 600 of 60 91 (148), 1 100 of 128 264 (372), 300 of 20
// 46 (69), 256 of 128 160 (116), 1 024 of 500 912 (834), 100 of 60 88 (43); bf16: 10 000 of 18 201 (471), 600 of 20 48 (45), 2 000 of 100
// 225 (253), 1 100 of 60 108 (87), 300 of 20 47 (36), 256 of 128 176 (52), 1 024 of 500 863 (396); 16 heads on 2 of 128, bf16: 10 000 of 18
// 757 (2 725), 600 of 20 119 (170), 2 000 of 100 972 (852).
bool few_rows(bool f32, int64_t tq, int64_t tk, int segments, int group) {
  const bool together = group == 1 || group == 2 || group == 4;
  const int64_t keys = together ? (segments >= 1024 ? 512 : segments >= 256 ? 128 : 64)
                                : (segments >= 512 ? (f32 ? 128 : 32) : f32 && segments >= 256 ? 32 : 0);
  return tq <= segments && tk <= keys * segments;
}

// Key splits of the forward: as many as bring the workgroups to one per CU, each with kSplitKeys keys at least of a
// segment of mean length. Their partial sums (dim + 2 floats a row) are joined by a second launch. Measured, us for one split,
// the taken number and twice as many: one query over 10 000 keys, fp32 245, 26 (19), 22; over 40 000, 16 heads on 4, bf16 538, 37
// (64), -; 16 such 616, 235 (4), 237; 2 000 rows of 1 head, fp32 55, 29 (3), 33; 2 000 rows of 8 heads of 64, bf16 28 (1), 40.
constexpr int kSplitKeys = 512, kSplitGroups = 256;

int split_count(bool f32, int dim, int64_t tq, int64_t tk, int segments, int heads, int kv_heads) {
  if (tq <= 0 || tk <= 0 || segments <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return 1;
  const int group = heads / kv_heads;
  if (few_rows(f32, tq, tk, segments, group)) return 1;
  const int rows = shape_rows(shape_of(f32, dim, tq * group, kv_heads, segments));
  const int64_t tiles = fmd_cdiv(fmd_cdiv(tq * group, segments), rows) * segments * kv_heads;
  const int64_t fill = kSplitGroups / tiles, most = tk / segments / kSplitKeys;
  const int64_t n = fill < most ? fill : most;
  return n < 1 ? 1 : n > kMaxSplits ? kMaxSplits : (int)n;
}

// Workspace, in floats from 16-byte aligned starts: the planes of two fp32 arrays of `rows` rows where the wide tiles take
// them, then the splits' partial sums.
int64_t planes_floats(int64_t rows, int heads, int dim) { return rows * heads * dim * 3; }  // two arrays of 3 bf16 planes

int64_t forward_floats(bool bf16, int splits, int64_t tq, int64_t tk, int segments, int heads, int kv_heads, int dim) {
  if (tq <= 0 || heads <= 0 || kv_heads <= 0 || dim <= 0 || heads % kv_heads) return 0;
  const bool planes = !bf16 && !few_rows(true, tq, tk, segments, heads / kv_heads) &&
                      shape_of(true, dim, tq * (heads / kv_heads), kv_heads, segments) != kNarrow;
  return (planes ? planes_floats(tk, kv_heads, dim) : 0) + (splits > 1 ? (int64_t)splits * tq * heads * (dim + 2) : 0);
}

// Splits of the VJP's walks, for as few workgroups: of the query rows for gk and gv, and of the keys for gq. Measured, us
// for one split, the taken number and twice as many: 2 000 causal rows of 8 heads on one of 128, bf16, gk and gv 303, 96 (4), 105;
// 2 000 rows of one head of 64, fp32, 75, 33 (4), 42 and gq 66, 35 (3), 40; 10 000 rows of 8 heads of 64, bf16, 689 (1), 725.
constexpr int kSplitRows = 256;

int row_splits(bool f32, int dim, int64_t tq, int64_t tk, int segments, int heads, int kv_heads) {
  const AttnShape shape = shape_of(f32, dim, tk, kv_heads, segments);
  if (segments <= 0) return 1;
  const int64_t tiles = fmd_cdiv(fmd_cdiv(tk, segments), shape_rows(shape)) * segments * kv_heads;
  const int64_t fill = tiles > 0 ? kSplitGroups / tiles : 1, most = tq * (heads / kv_heads) / segments / kSplitRows;
  const int64_t n = fill < most ? fill : most;
  return n < 1 ? 1 : n > kMaxSplits ? kMaxSplits : (int)n;
}

int64_t backward_floats(bool bf16, int64_t tq, int64_t tk, int segments, int heads, int kv_heads, int dim, int q_splits,
                        int kv_splits) {
  if (heads <= 0 || kv_heads <= 0 || dim <= 0 || heads % kv_heads || tq < 0 || tk < 0) return 0;
  int64_t n = fmd_cdiv(2 * heads * tq, 4) * 4;  // offsets and deltas
  if (few_rows(!bf16, tq, tk, segments, heads / kv_heads)) return n;
  if (!bf16) {
    if (shape_of(true, dim, tq * (heads / kv_heads), kv_heads, segments) != kNarrow) n += planes_floats(tk, kv_heads, dim);
    if (shape_of(true, dim, tk, kv_heads, segments) != kNarrow) n += planes_floats(tq, heads, dim);
  }
  if (q_splits > 1) n += q_splits * tq * heads * dim;
  if (kv_splits > 1) n += kv_splits * 2 * tk * kv_heads * dim;
  return n;
}

// the planes of two arrays, formed into `work`, which moves past them
int split_planes(const void* x, int64_t x_row, int64_t x_head, const void* y, int64_t y_row, int64_t y_head, int64_t rows, int heads,
                 int dim, float*& work, AttnTiles* t, hipStream_t stream) {
  __bf16* xp = reinterpret_cast<__bf16*>(work);
  __bf16* yp = xp + rows * heads * dim * 3;
  work += planes_floats(rows, heads, dim);
  const int64_t ld = (int64_t)heads * dim * 3;
  *t = {xp, yp, ld, 3 * dim, ld, 3 * dim};
  const int64_t n = rows * heads * (dim / 8);
  if (n == 0) return FMD_OK;
  FMD_REQUIRE(ld < (1 << 24) && n < (1ll << 32));
  attn_split_kernel<<<(unsigned)fmd_cdiv(n, 256), 256, 0, stream>>>(static_cast<const float*>(x), x_row, x_head,
                                                                    static_cast<const float*>(y), y_row, y_head, rows, heads, dim, xp, yp);
  FMD_CHECK_LAUNCH();
  return FMD_OK;
}

AttnTiles bf16_tiles(const void* x, int64_t x_row, int64_t x_head, const void* y, int64_t y_row, int64_t y_head) {
  return {static_cast<const __bf16*>(x), static_cast<const __bf16*>(y), x_row, x_head, y_row, y_head};
}

template <typename T, int DP, bool CAUSAL>
int run_fwd(const AttnArgs& a, int splits, T* out, const AttnSaved& saved, float* work, hipStream_t stream) {
  constexpr bool f32 = AttnType<T>::planes == 3;
  // Keys of a wide tile: 64 (4 x 3 000 rows, 8 heads, bf16: 182 us against 221 of 32 keys at 96 columns, 161 against 170 at 64, 219
  // against 222 at 128; causal, 16 heads of 128: one segment of 4 000 rows 130 against 143, five prompts of 12 000 together 337 against
  // 332; fp32 at 32: 234 against 282), but 32 where more has no registers (fp32 above 32).
  constexpr int kKeyWaves = f32 && DP > 64 ? 2 : 4, kWideKeys = f32 && DP > 32 ? 32 : 64;
  const int64_t n = a.tq * a.heads;
  AttnTiles t = bf16_tiles(a.k, a.k_row, a.k_head, a.v, a.v_row, a.v_head);
  const AttnShape shape = shape_of(f32, a.dim, a.tq * a.group, a.kv_heads, a.segments);
  FMD_REQUIRE(work || (splits == 1 && !(f32 && shape != kNarrow && a.tk > 0)));
  if (f32 && shape != kNarrow) {
    const int status = split_planes(a.k, a.k_row, a.k_head, a.v, a.v_row, a.v_head, a.tk, a.kv_heads, a.dim, work, &t, stream);
    if (status != FMD_OK) return status;
  }
  float *po = work, *pm = work ? work + splits * n * a.dim : nullptr, *pl = work ? pm + splits * n : nullptr;
  const int64_t tiles = tile_count(a.tq, a.group, a.segments, shape_rows(shape));
  const int status = launch_ranges(tiles * a.kv_heads, [&](unsigned blocks, int64_t first) {
    const dim3 grid(blocks, splits);
    AttnArgs b = a;
    b.block0 = (uint32_t)first;
    if (shape == kWide) {
      attn_fwd_kernel<T, DP, kWideKeys, 4, 1, true, CAUSAL><<<grid, 256, 0, stream>>>(b, t, tiles, splits, out, saved, po, pm, pl);
    } else if (shape == kMid) {
      if constexpr (f32 && DP <= 64)
        attn_fwd_kernel<T, DP, 32, 2, 2, true, CAUSAL><<<grid, 256, 0, stream>>>(b, t, tiles, splits, out, saved, po, pm, pl);
    } else {
      attn_fwd_kernel<T, DP, 32, 1, kKeyWaves, !f32, CAUSAL><<<grid, 64 * kKeyWaves, 0, stream>>>(b, t, tiles, splits, out, saved, po, pm, pl);
    }
  });
  if (status != FMD_OK) return status;
  if (splits > 1) {  // of calls with too few tiles to fill the card: few rows
    attn_join_kernel<T><<<(unsigned)fmd_cdiv(n, 4), 256, 0, stream>>>(a, splits, po, pm, pl, out, saved);
    FMD_CHECK_LAUNCH();
  }
  return FMD_OK;
}

template <typename T, int DP, bool CAUSAL>
int run_bwd(const AttnArgs& a, const AttnBwd& b, int q_splits, int kv_splits, T* gq, T* gk, T* gv, float* work, hipStream_t stream) {
  constexpr bool f32 = AttnType<T>::planes == 3;
  constexpr int kWaves = f32 && DP > 64 ? 2 : 4;
  if (gk) {
    AttnTiles t = bf16_tiles(a.q, a.q_row, a.q_head, b.g, b.g_row, b.g_head);
    const AttnShape shape = shape_of(f32, a.dim, a.tk, a.kv_heads, a.segments);
    if (f32 && shape != kNarrow) {
      const int status = split_planes(a.q, a.q_row, a.q_head, b.g, b.g_row, b.g_head, a.tq, a.heads, a.dim, work, &t, stream);
      if (status != FMD_OK) return status;
    }
    // wide bf16: 64 keys and four row groups, two waves per SIMD in one workgroup
    constexpr int kWM = f32 ? 4 : 2, kRW = f32 ? 1 : 4, kMidRW = DP <= 32 ? 4 : 2;
    const int64_t tiles = tile_count(a.tk, 1, a.segments, shape == kWide ? 32 * kWM : shape_rows(shape));
    float* part = work;
    if (kv_splits > 1) work += kv_splits * 2 * a.tk * a.kv_heads * a.dim;
    const int status = launch_ranges(tiles * a.kv_heads, [&](unsigned blocks, int64_t first) {
      const dim3 grid(blocks, kv_splits);
      AttnArgs c = a;
      c.block0 = (uint32_t)first;
      if (shape == kWide) {
        attn_bwd_kv_kernel<T, DP, kWM, kRW, true, CAUSAL><<<grid, 64 * kWM * kRW, 0, stream>>>(c, b, t, kv_splits, part, gk, gv);
      } else if (shape == kMid) {
        if constexpr (f32 && DP <= 64)
          attn_bwd_kv_kernel<T, DP, 2, kMidRW, true, CAUSAL><<<grid, 128 * kMidRW, 0, stream>>>(c, b, t, kv_splits, part, gk, gv);
      } else {
        attn_bwd_kv_kernel<T, DP, 1, kWaves, !f32, CAUSAL><<<grid, 64 * kWaves, 0, stream>>>(c, b, t, kv_splits, part, gk, gv);
      }
    });
    if (status != FMD_OK) return status;
    if (kv_splits > 1) {
      const int64_t n = a.tk * a.kv_heads * a.dim;
      attn_add_kernel<T><<<(unsigned)fmd_cdiv(2 * n, 1024), 256, 0, stream>>>(part, n, kv_splits, gk, gv);
      FMD_CHECK_LAUNCH();
    }
  }
  if (gq) {
    AttnTiles t = bf16_tiles(a.k, a.k_row, a.k_head, a.v, a.v_row, a.v_head);
    const AttnShape shape = shape_of(f32, a.dim, a.tq * a.group, a.kv_heads, a.segments);
    if (f32 && shape != kNarrow) {
      const int status = split_planes(a.k, a.k_row, a.k_head, a.v, a.v_row, a.v_head, a.tk, a.kv_heads, a.dim, work, &t, stream);
      if (status != FMD_OK) return status;
    }
    const int64_t tiles = tile_count(a.tq, a.group, a.segments, shape_rows(shape));
    float* part = work;
    const int status = launch_ranges(tiles * a.kv_heads, [&](unsigned blocks, int64_t first) {
      const dim3 grid(blocks, q_splits);
      AttnArgs c = a;
      c.block0 = (uint32_t)first;
      if (shape == kWide) {
        attn_bwd_q_kernel<T, DP, 4, 1, true, CAUSAL><<<grid, 256, 0, stream>>>(c, b, t, tiles, q_splits, part, gq);
      } else if (shape == kMid) {
        if constexpr (f32 && DP <= 64) attn_bwd_q_kernel<T, DP, 2, 2, true, CAUSAL><<<grid, 256, 0, stream>>>(c, b, t, tiles, q_splits, part, gq);
      } else {
        attn_bwd_q_kernel<T, DP, 1, kWaves, !f32, CAUSAL><<<grid, 64 * kWaves, 0, stream>>>(c, b, t, tiles, q_splits, part, gq);
      }
    });
    if (status != FMD_OK) return status;
    if (q_splits > 1) {
      const int64_t n = a.tq * a.heads * a.dim;
      attn_add_kernel<T><<<(unsigned)fmd_cdiv(n, 1024), 256, 0, stream>>>(part, n, q_splits, gq, static_cast<T*>(nullptr));
      FMD_CHECK_LAUNCH();
    }
  }
  return FMD_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// what the kernels' 16-byte loads and index arithmetic assume
int check(const AttnArgs& a, int size) {
  FMD_REQUIRE(a.tq >= 0 && a.tk >= 0 && a.segments >= 0 && a.heads > 0 && a.kv_heads > 0 && a.dim > 0);
  FMD_REQUIRE(a.heads % a.kv_heads == 0 && a.q_off && a.k_off);
  FMD_REQUIRE(a.tq * a.group < (1ll << 31) && a.tk < (1ll << 31) && a.segments < (1 << 30));
  if (a.dim > 128 || a.dim % 8 != 0) return FMD_EUNSUPPORTED;
  FMD_REQUIRE((a.q || a.tq == 0) && (a.tk == 0 || (a.k && a.v)));
  const int64_t unit = 16 / size;
  FMD_REQUIRE(aligned16(a.q) && aligned16(a.k) && aligned16(a.v));
  FMD_REQUIRE(a.q_row % unit == 0 && a.q_head % unit == 0 && a.k_row % unit == 0 && a.k_head % unit == 0 &&
              a.v_row % unit == 0 && a.v_head % unit == 0);
  FMD_REQUIRE(a.q_row < (1 << 24) && a.k_row < (1 << 24) && a.v_row < (1 << 24));
  FMD_REQUIRE(a.scale > 0.f);
  // workgroups are numbered in 32 bits
  FMD_REQUIRE((std::max(a.tq * a.group, a.tk) / 32 + a.segments + 2) * a.kv_heads < (1ll << 31));
  return FMD_OK;
}

#define FMD_BY_WIDTH(F, ...)                                                                    \
  if (a.dim <= 32) return a.causal ? F<T, 32, true>(__VA_ARGS__) : F<T, 32, false>(__VA_ARGS__); \
  if (a.dim <= 64) return a.causal ? F<T, 64, true>(__VA_ARGS__) : F<T, 64, false>(__VA_ARGS__); \
  if (a.dim <= 96) return a.causal ? F<T, 96, true>(__VA_ARGS__) : F<T, 96, false>(__VA_ARGS__); \
  return a.causal ? F<T, 128, true>(__VA_ARGS__) : F<T, 128, false>(__VA_ARGS__);

template <typename T>
int forward(const AttnArgs& a, int splits, T* out, const AttnSaved& saved, float* work, hipStream_t stream) {
  const int status = check(a, sizeof(T));
  if (status != FMD_OK) return status;
  FMD_REQUIRE(splits >= 1 && splits <= kMaxSplits && aligned16(work));
  if (a.tq == 0) return FMD_OK;
  FMD_REQUIRE(out && aligned16(out) && aligned16(saved.residual) && (saved.base == nullptr) == (saved.inverse == nullptr));
  if (few_rows(sizeof(T) == 4, a.tq, a.tk, a.segments, a.group)) return attn_rows_fwd<T>(a, out, saved, stream);
  FMD_BY_WIDTH(run_fwd, a, splits, out, saved, work, stream)
}

template <typename T>
int backward(const AttnArgs& a, AttnBwd b, int q_splits, int kv_splits, T* gq, T* gk, T* gv, float* work, hipStream_t stream) {
  const int status = check(a, sizeof(T));
  if (status != FMD_OK) return status;
  const int64_t unit = 16 / sizeof(T);
  FMD_REQUIRE(a.tq == 0 || (b.g && b.out && b.saved.base && b.saved.inverse && (sizeof(T) == 4 || b.saved.residual)));
  FMD_REQUIRE(aligned16(b.g) && aligned16(b.out) && aligned16(b.saved.residual));
  FMD_REQUIRE(b.g_row % unit == 0 && b.g_head % unit == 0);
  FMD_REQUIRE((gk == nullptr) == (gv == nullptr) && aligned16(gq) && aligned16(gk) && aligned16(gv));
  FMD_REQUIRE(q_splits >= 1 && q_splits <= kMaxSplits && kv_splits >= 1 && kv_splits <= kMaxSplits);
  FMD_REQUIRE(work && aligned16(work));
  b.rows = work;
  if (a.tq == 0) gq = nullptr;
  if (a.tk == 0) gk = gv = nullptr;
  if (few_rows(sizeof(T) == 4, a.tq, a.tk, a.segments, a.group)) return attn_rows_bwd<T>(a, b, gq, gk, gv, stream);
  if (a.tq > 0) {
    const int launched = launch_ranges(fmd_cdiv(a.tq * a.heads, 16), [&](unsigned blocks, int64_t first) {
      attn_delta_kernel<T><<<blocks, 256, 0, stream>>>(b, a.tq, a.heads, a.dim, first, work);
    });
    if (launched != FMD_OK) return launched;
  }
  work += fmd_cdiv(2 * a.heads * a.tq, 4) * 4;
  FMD_BY_WIDTH(run_bwd, a, b, q_splits, kv_splits, gq, gk, gv, work, stream)
}

AttnArgs args_of(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v,
                 int64_t v_row, int64_t v_head, const int64_t* q_off, const int64_t* k_off, int64_t tq, int64_t tk,
                 int32_t segments, int32_t heads, int32_t kv_heads, int32_t dim, int32_t causal, float scale) {
  AttnArgs a = {};
  a.q = q, a.k = k, a.v = v;
  a.q_row = q_row, a.q_head = q_head, a.k_row = k_row, a.k_head = k_head, a.v_row = v_row, a.v_head = v_head;
  a.q_off = q_off, a.k_off = k_off, a.tq = tq, a.tk = tk;
  a.segments = segments, a.heads = heads, a.kv_heads = kv_heads, a.group = kv_heads > 0 ? heads / kv_heads : 0;
  a.dim = dim, a.causal = causal, a.scale = scale;
  // ceil(2^(31 + s) / group) with group <= 2^s: exact for rows below 2^31
  while ((1ll << (a.group_shift)) < a.group) ++a.group_shift;
  a.group_shift += 31;
  a.group_mul = a.group > 0 ? (uint32_t)(((1ull << a.group_shift) + a.group - 1) / a.group) : 0;
  return a;
}

}  // namespace

extern "C" {

#define FMD_ATTN_PARAMS                                                                                          \
  const void *q, int64_t q_row, int64_t q_head, const void *k, int64_t k_row, int64_t k_head, const void *v,     \
      int64_t v_row, int64_t v_head, const int64_t *q_offsets, const int64_t *k_offsets, int64_t tq, int64_t tk, \
      int32_t segments, int32_t heads, int32_t kv_heads, int32_t dim, int32_t causal, float scale
#define FMD_ATTN_ARGS                                                                                            \
  args_of(q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, q_offsets, k_offsets, tq, tk, segments, heads,   \
          kv_heads, dim, causal, scale)

int32_t fmd_segment_attention_splits(int32_t bf16, int64_t tq, int64_t tk, int32_t segments, int32_t heads, int32_t kv_heads,
                                     int32_t dim) {
  return split_count(!bf16, dim, tq, tk, segments, heads, kv_heads);
}

int64_t fmd_segment_attention_work_size(int32_t bf16, int32_t splits, int64_t tq, int64_t tk, int32_t segments, int32_t heads,
                                        int32_t kv_heads, int32_t dim) {
  return forward_floats(bf16, splits, tq, tk, segments, heads, kv_heads, dim);
}

int32_t fmd_segment_attention_bwd_splits(int32_t bf16, int64_t tq, int64_t tk, int32_t segments, int32_t heads, int32_t kv_heads,
                                         int32_t dim, int32_t of_kv) {
  if (tq <= 0 || tk <= 0 || segments <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return 1;
  if (few_rows(!bf16, tq, tk, segments, heads / kv_heads)) return 1;
  return of_kv ? row_splits(!bf16, dim, tq, tk, segments, heads, kv_heads)
               : split_count(!bf16, dim, tq, tk, segments, heads, kv_heads);
}

int64_t fmd_segment_attention_bwd_work_size(int32_t bf16, int64_t tq, int64_t tk, int32_t segments, int32_t heads,
                                            int32_t kv_heads, int32_t dim, int32_t q_splits, int32_t kv_splits) {
  return backward_floats(bf16, tq, tk, segments, heads, kv_heads, dim, q_splits, kv_splits);
}

int fmd_segment_attention(int32_t bf16, FMD_ATTN_PARAMS, int32_t splits, void* out, float* base, float* inverse,
                          void* residual, float* work, hipStream_t stream) {
  const AttnArgs a = FMD_ATTN_ARGS;
  const AttnSaved saved = {base, inverse, bf16 ? residual : nullptr};
  return bf16 ? forward(a, splits, static_cast<__bf16*>(out), saved, work, stream)
              : forward(a, splits, static_cast<float*>(out), saved, work, stream);
}

int fmd_segment_attention_bwd(int32_t bf16, FMD_ATTN_PARAMS, const void* gout, int64_t g_row, int64_t g_head, const void* out,
                              const float* base, const float* inverse, const void* residual, int32_t q_splits, int32_t kv_splits,
                              float* work, void* gq, void* gk, void* gv, hipStream_t stream) {
  const AttnArgs a = FMD_ATTN_ARGS;
  const AttnSaved saved = {const_cast<float*>(base), const_cast<float*>(inverse), const_cast<void*>(residual)};
  const AttnBwd b = {gout, g_row, g_head, out, saved, nullptr};
  return bf16 ? backward(a, b, q_splits, kv_splits, static_cast<__bf16*>(gq), static_cast<__bf16*>(gk), static_cast<__bf16*>(gv), work, stream)
              : backward(a, b, q_splits, kv_splits, static_cast<float*>(gq), static_cast<float*>(gk), static_cast<float*>(gv), work, stream);
}

}  // extern "C"
