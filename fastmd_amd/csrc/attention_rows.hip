// Segment attention of about one query per segment over a few keys each (an atom over its neighbour rows), and its VJP:
// memory-bound, on the vector units, in fp32.
//
// One wave per segment and block of key heads, but for long segments (attn_long): a wave's work is bounded whatever the offsets
// are (2 048 slots, one of 1 500 queries over as many keys, 4 heads of 32, fp32: 0.95 ms forward, 2.5 VJP). A unit of D / 8 lanes (a power of two) takes one key row of one head, eight
// columns a lane; the units of a wave lie along the heads (a row's heads are contiguous) and then along keys. Every key row is
// read once and, in the VJP of a single query, its two gradients are written in the same pass. The matrix kernels spend a
// tile of 32 rows on such a segment's single one. 10 000 segments, 180 096 keys, 4 heads of 32: 35 + 75 us forward and VJP in
// float32 (195 and 389 MB: 5.6 and 5.1 TB/s, where a large copy reaches 4.8, the caches holding part of it; 1 004 us on the
// matrix kernels), 20 + 34 us in bf16.
#include "attention.h"

namespace {

__device__ __forceinline__ void zero8(float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
}

__device__ __forceinline__ float dot8(const float (&x)[8], const float (&y)[8]) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = fmaf(x[i], y[i], s);
  return s;
}

// a wave's place: head block, and the lane's unit
struct RowLane {
  int col, kvh, slot, slots, stride;  // stride: lanes from one key slot to the next
  bool on;                            // the lane has columns of a head
};

template <int LG>
__device__ __forceinline__ RowLane row_lane(const AttnArgs& a, int head_block, int hb) {
  const int lane = threadIdx.x & 63, unit = lane / LG;
  RowLane r;
  r.col = 8 * (lane & (LG - 1));
  r.kvh = head_block * hb + unit % hb;
  r.slot = unit / hb;
  r.slots = 64 / LG / hb;
  r.stride = LG * hb;
  r.on = r.col < a.dim && r.kvh < a.kv_heads;
  if (!r.on) r.kvh = 0;
  return r;
}

// The extended segment of wave w: the caller's segments first, then kTail waves that clear the rows outside them.
constexpr int kTail = 64;

// rows outside every segment, dealt out over the tail waves: [0, first offset) and [last offset, rows)
template <typename T>
__device__ __forceinline__ void clear_outside(const int64_t* off, int segments, int64_t rows, int width, int tail, T* x, float* base,
                                              float* inverse, int heads) {
  const int lane = threadIdx.x & 63;
  const int64_t lo = attn_start(off, segments, rows, 1), hi = attn_start(off, segments, rows, segments + 1);
  for (int64_t n = tail; n < lo + rows - hi; n += kTail) {
    const int64_t row = n < lo ? n : hi + n - lo;
    for (int c = lane; c < width; c += 64) x[row * width + c] = (T)0.f;
    if (base)
      for (int h = lane; h < heads; h += 64) base[h * rows + row] = inverse[h * rows + row] = 0.f;
  }
}

// One query row over the keys first, first + step, ... below `sees`, for G heads of its group: their weighted values, maxima and sums,
// joined over the wave's key slots.
template <typename T, int LG, int G>
struct RowSoftmax {
  float o[G][8], m[G], l[G];

  __device__ __forceinline__ void walk(const AttnArgs& a, const RowLane& r, const AttnSegment& sg, int i, int head, uint32_t first,
                                       uint32_t step) {
    const uint32_t sees = a.causal ? max(0, min(sg.nk, i + sg.nk - sg.nq + 1)) : sg.nk;
    const float c = a.scale * kLog2e;
    const T* kb = static_cast<const T*>(a.k) + sg.k0 * a.k_row + r.kvh * a.k_head + r.col;
    const T* vb = static_cast<const T*>(a.v) + sg.k0 * a.v_row + r.kvh * a.v_head + r.col;
    const T* qp = static_cast<const T*>(a.q) + (sg.q0 + i) * a.q_row + head * a.q_head + r.col;
    float q[G][8];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      zero8(q[g]);
      zero8(o[g]);
      if (r.on) load8<T>(qp + g * a.q_head, q[g]);
      m[g] = -INFINITY;
      l[g] = 0.f;
    }
    for (uint32_t j = first; j < sees; j += step) {
      float k[8], v[8];
      zero8(k);
      zero8(v);
      if (r.on) {
        load8<T>(kb + j * a.k_row, k);
        load8<T>(vb + j * a.v_row, v);
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float s = lanes_sum<LG>(dot8(q[g], k)) * c;
        const float top = fmaxf(m[g], s), shift = top == -INFINITY ? 0.f : top;
        const float fade = exp2_hw(m[g] - shift), p = exp2_hw(s - shift);
        l[g] = fmaf(l[g], fade, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[g][e] = fmaf(o[g][e], fade, p * v[e]);
        m[g] = top;
      }
    }
    for (int by = r.stride; by < 64; by *= 2) {  // the key slots of a head
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float oo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) oo[e] = __shfl_xor(o[g][e], by, 64);
        const float om = __shfl_xor(m[g], by, 64), ol = __shfl_xor(l[g], by, 64);
        join(g, om, ol, oo);
      }
    }
  }

  __device__ __forceinline__ void join(int g, float om, float ol, const float (&oo)[8]) {
    const float top = fmaxf(m[g], om), shift = top == -INFINITY ? 0.f : top;
    const float fa = exp2_hw(m[g] - shift), fb = exp2_hw(om - shift);
    l[g] = l[g] * fa + ol * fb;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[g][e] = o[g][e] * fa + oo[e] * fb;
    m[g] = top;
  }

  __device__ __forceinline__ void store(const AttnArgs& a, const RowLane& r, int64_t row, int head, int g, T* out, const AttnSaved& saved) {
    const float inv = l[g] > 0.f || l[g] != l[g] ? 1.f / l[g] : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[g][e] *= inv;
    const int64_t at = (row * a.heads + head + g) * a.dim + r.col;
    store8<false>(out + at, o[g]);
    saved_residual<T>(saved, at, o[g]);
    if (saved.base && r.col == 0) {
      const int64_t s = (head + g) * a.tq + row;
      saved.base[s] = m[g] == -INFINITY ? 0.f : m[g];
      saved.inverse[s] = inv;
    }
  }
};

// The part of a long segment that a workgroup past the `row_blocks` takes: its queries part, part + parts, ..., with the keys of each dealt
// out to its four waves.
struct LongPart {
  AttnSegment sg;
  int64_t part, parts;
  int head_block;
  bool any;
};

__device__ __forceinline__ LongPart long_part(const AttnArgs& a, int64_t number, int head_blocks) {
  LongPart p;
  p.head_block = (int)(number % head_blocks);
  const int i = attn_share(a.q_off, a.k_off, a.segments, a.tq, a.tk, number / head_blocks, &p.part, &p.parts, WaveLanes());
  p.sg = attn_segment(a, i);
  p.any = attn_real(a, i) && attn_long(p.sg.nq, p.sg.nk) && p.part < p.parts;
  return p;
}

// GF: query heads taken together (the whole group); 0: one after the other, with a walk over the keys each
template <typename T, int LG, int GF>
__global__ void __launch_bounds__(256) attn_rows_fwd_kernel(AttnArgs a, int hb, int head_blocks, int64_t row_blocks, T* out, AttnSaved saved) {
  constexpr int G = GF ? GF : 1;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  RowSoftmax<T, LG, G> x;
  const int64_t block = (int64_t)a.block0 + blockIdx.x;
  if (block >= row_blocks) {
    __shared__ float part[3][10][64];
    const LongPart p = long_part(a, block - row_blocks, head_blocks);
    if (!p.any) return;
    const RowLane r = row_lane<LG>(a, p.head_block, hb);
    for (int64_t i = p.part; i < p.sg.nq; i += p.parts)
      for (int g0 = 0; g0 < a.group; g0 += G) {
        const int head = r.kvh * a.group + g0;
        x.walk(a, r, p.sg, (int)i, head, wave * r.slots + r.slot, 4 * r.slots);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          __syncthreads();  // the part before is read
          if (wave > 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) part[wave - 1][e][lane] = x.o[g][e];
            part[wave - 1][8][lane] = x.m[g];
            part[wave - 1][9][lane] = x.l[g];
          }
          __syncthreads();
          if (wave == 0) {
            for (int n = 0; n < 3; ++n) {
              float o[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) o[e] = part[n][e][lane];
              x.join(g, part[n][8][lane], part[n][9][lane], o);
            }
            if (r.on && r.slot == 0) x.store(a, r, p.sg.q0 + i, head, g, out, saved);
          }
        }
      }
    return;
  }
  const int64_t w = block * 4 + wave;
  const int64_t seg = w / head_blocks;
  const RowLane r = row_lane<LG>(a, (int)(w % head_blocks), hb);
  if (seg >= a.segments) {
    if (seg - a.segments < kTail && w % head_blocks == 0)
      clear_outside(a.q_off, a.segments, a.tq, a.heads * a.dim, (int)(seg - a.segments), out, saved.base, saved.inverse, a.heads);
    return;
  }
  const AttnSegment sg = attn_segment(a, (int)seg + 1);
  if (attn_long(sg.nq, sg.nk)) return;
  for (int i = 0; i < sg.nq; ++i)
    for (int g0 = 0; g0 < a.group; g0 += G) {
      const int head = r.kvh * a.group + g0;
      x.walk(a, r, sg, i, head, r.slot, r.slots);
      if (r.on && r.slot == 0) {
#pragma unroll
        for (int g = 0; g < G; ++g) x.store(a, r, sg.q0 + i, head, g, out, saved);
      }
    }
}

// sum of x over the lanes of all key slots
__device__ __forceinline__ void slots_sum(float (&x)[8], int stride) {
  for (int by = stride; by < 64; by *= 2)
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] += __shfl_xor(x[e], by, 64);
}

template <typename T>
__device__ __forceinline__ float delta_part(const AttnBwd& b, int64_t at, const float (&g)[8]) {
  float o[8];
  load8<T>(static_cast<const T*>(b.out) + at, o);
  float s = dot8(o, g);
  if constexpr (sizeof(T) == 2) {
    load8<T>(static_cast<const T*>(b.saved.residual) + at, o);
    s += dot8(o, g);
  }
  return s;
}

// GF: the group, for segments of one query: one pass over the keys forms all three gradients. A segment of another
// number of queries, and GF = 0, takes a pass per query head for gq and one for gk and gv, whose sums run over all of
// them in order; so do the parts of a long segment.
template <typename T, int LG, int GF, bool NT>
__global__ void __launch_bounds__(256) attn_rows_bwd_kernel(AttnArgs a, AttnBwd b, int hb, int head_blocks, int64_t row_blocks, T* gq, T* gk,
                                                            T* gv) {
  constexpr int G = GF ? GF : 1;
  const int64_t block = (int64_t)a.block0 + blockIdx.x;
  const bool is_long = block >= row_blocks;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int64_t part = 0, parts = 1;
  AttnSegment sg;
  RowLane r;
  if (is_long) {
    const LongPart p = long_part(a, block - row_blocks, head_blocks);
    if (!p.any) return;
    sg = p.sg;
    part = p.part;
    parts = p.parts;
    r = row_lane<LG>(a, p.head_block, hb);
  } else {
    const int64_t w = block * 4 + wave;
    const int64_t seg = w / head_blocks;
    r = row_lane<LG>(a, (int)(w % head_blocks), hb);
    if (seg >= a.segments) {
      if (seg - a.segments < kTail && w % head_blocks == 0) {
        const int tail = (int)(seg - a.segments);
        if (gq) clear_outside<T>(a.q_off, a.segments, a.tq, a.heads * a.dim, tail, gq, nullptr, nullptr, 0);
        if (gk) {
          clear_outside<T>(a.k_off, a.segments, a.tk, a.kv_heads * a.dim, tail, gk, nullptr, nullptr, 0);
          clear_outside<T>(a.k_off, a.segments, a.tk, a.kv_heads * a.dim, tail, gv, nullptr, nullptr, 0);
        }
      }
      return;
    }
    sg = attn_segment(a, (int)seg + 1);
    if (attn_long(sg.nq, sg.nk)) return;
  }
  const float c = a.scale * kLog2e;
  const T* kb = static_cast<const T*>(a.k) + sg.k0 * a.k_row + r.kvh * a.k_head + r.col;
  const T* vb = static_cast<const T*>(a.v) + sg.k0 * a.v_row + r.kvh * a.v_head + r.col;
  const int64_t kat = (sg.k0 * a.kv_heads + r.kvh) * a.dim + r.col, kstep = (int64_t)a.kv_heads * a.dim;
  // one query row of one head: its columns, statistics and delta
  struct Query {
    float q[8], g[8], base, inv, delta;
  };
  auto query = [&](int i, int head, Query& x) {
    zero8(x.q);
    zero8(x.g);
    float d = 0.f;
    if (r.on) {
      load8<T>(static_cast<const T*>(a.q) + (sg.q0 + i) * a.q_row + head * a.q_head + r.col, x.q);
      load8<T>(static_cast<const T*>(b.g) + (sg.q0 + i) * b.g_row + head * b.g_head + r.col, x.g);
      d = delta_part<T>(b, ((sg.q0 + i) * a.heads + head) * a.dim + r.col, x.g);
    }
    x.delta = lanes_sum<LG>(d);
    x.inv = b.saved.inverse[head * a.tq + sg.q0 + i];
    x.base = x.inv == 0.f ? INFINITY : b.saved.base[head * a.tq + sg.q0 + i];
  };
  auto sees = [&](int i) { return a.causal ? max(0, min(sg.nk, i + sg.nk - sg.nq + 1)) : sg.nk; };
  auto weights = [&](const Query& x, const float (&k)[8], const float (&v)[8], float& p, float& ds) {
    const float s = lanes_sum<LG>(dot8(x.q, k)), dp = lanes_sum<LG>(dot8(x.g, v));
    p = exp2_hw(fmaf(s, c, -x.base)) * x.inv;
    ds = p * (dp - x.delta) * a.scale;
  };

  if (GF && sg.nq == 1 && !is_long) {
    Query x[G];
    float dq[G][8];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      query(0, r.kvh * a.group + g, x[g]);
      zero8(dq[g]);
    }
    for (int j = r.slot; j < sg.nk; j += r.slots) {
      float k[8], v[8], dk[8], dv[8];
      zero8(k);
      zero8(v);
      zero8(dk);
      zero8(dv);
      if (r.on) {
        load8<T>(kb + j * a.k_row, k);
        load8<T>(vb + j * a.v_row, v);
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float p, ds;
        weights(x[g], k, v, p, ds);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dk[e] = fmaf(ds, x[g].q[e], dk[e]);
          dv[e] = fmaf(p, x[g].g[e], dv[e]);
          dq[g][e] = fmaf(ds, k[e], dq[g][e]);
        }
      }
      if (r.on && gk) {
        store8<NT>(gk + kat + j * kstep, dk);
        store8<NT>(gv + kat + j * kstep, dv);
      }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      slots_sum(dq[g], r.stride);
      if (r.on && r.slot == 0 && gq) store8<false>(gq + (sg.q0 * a.heads + r.kvh * a.group + g) * a.dim + r.col, dq[g]);
    }
    return;
  }
  // the walk's first key and step: the wave's slots, or the workgroup's
  const uint32_t waves = is_long ? 4 : 1, place = is_long ? wave : 0;
  if (gq)
    for (int64_t i = part; i < sg.nq; i += parts)
      for (int g = 0; g < a.group; ++g) {
        const int head = r.kvh * a.group + g;
        const uint32_t n = sees((int)i);
        Query x;
        query((int)i, head, x);
        float dq[8];
        zero8(dq);
        for (uint32_t j = place * r.slots + r.slot; j < n; j += waves * r.slots) {
          float k[8], v[8], p, ds;
          zero8(k);
          zero8(v);
          if (r.on) {
            load8<T>(kb + j * a.k_row, k);
            load8<T>(vb + j * a.v_row, v);
          }
          weights(x, k, v, p, ds);
#pragma unroll
          for (int e = 0; e < 8; ++e) dq[e] = fmaf(ds, k[e], dq[e]);
        }
        slots_sum(dq, r.stride);
        if (is_long) {
          __shared__ float sum[3][8][64];
          __syncthreads();  // the sum before is read
          if (wave > 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[wave - 1][e][lane] = dq[e];
          }
          __syncthreads();
          for (int k = 0; k < 3; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) dq[e] += sum[k][e][lane];  // of the first wave's use alone
        }
        if (r.on && r.slot == 0 && place == 0) store8<false>(gq + ((sg.q0 + i) * a.heads + head) * a.dim + r.col, dq);
      }
  if (!gk) return;
  for (int64_t j0 = (part * waves + place) * r.slots; j0 < sg.nk; j0 += parts * waves * r.slots) {
    const int64_t j = j0 + r.slot;
    const bool live = r.on && j < sg.nk;
    float k[8], v[8], dk[8], dv[8];
    zero8(k);
    zero8(v);
    zero8(dk);
    zero8(dv);
    if (live) {
      load8<T>(kb + j * a.k_row, k);
      load8<T>(vb + j * a.v_row, v);
    }
    for (int i = 0; i < sg.nq; ++i)
      for (int g = 0; g < a.group; ++g) {
        Query x;
        query(i, r.kvh * a.group + g, x);
        float p, ds;
        weights(x, k, v, p, ds);
        if (j >= sees(i)) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dk[e] = fmaf(ds, x.q[e], dk[e]);
          dv[e] = fmaf(p, x.g[e], dv[e]);
        }
      }
    if (live) {
      store8<NT>(gk + kat + j * kstep, dk);
      store8<NT>(gv + kat + j * kstep, dv);
    }
  }
}

int pow2_at_least(int x) {
  int p = 1;
  while (p < x) p *= 2;
  return p;
}

struct RowGrid {
  int hb, head_blocks;
  int64_t row_blocks, blocks;
};

RowGrid row_grid(const AttnArgs& a, int lg) {
  RowGrid r;
  const int most = 64 / lg, want = pow2_at_least(a.kv_heads);
  r.hb = want < most ? want : most;
  r.head_blocks = (int)fmd_cdiv(a.kv_heads, r.hb);
  r.row_blocks = fmd_cdiv(((int64_t)a.segments + kTail) * r.head_blocks, 4);
  r.blocks = r.row_blocks + attn_long_numbers(a.tq, a.tk) * r.head_blocks;
  return r;
}

template <typename T, int LG>
int fwd(const AttnArgs& a, T* out, const AttnSaved& s, hipStream_t stream) {
  const RowGrid r = row_grid(a, LG);
  FMD_REQUIRE(r.blocks < (1ll << 32));
  return launch_ranges(r.blocks, [&](unsigned n, int64_t first) {
    AttnArgs c = a;
    c.block0 = (uint32_t)first;
    if (a.group == 1) attn_rows_fwd_kernel<T, LG, 1><<<n, 256, 0, stream>>>(c, r.hb, r.head_blocks, r.row_blocks, out, s);
    else if (a.group == 2) attn_rows_fwd_kernel<T, LG, 2><<<n, 256, 0, stream>>>(c, r.hb, r.head_blocks, r.row_blocks, out, s);
    else if (a.group == 4) attn_rows_fwd_kernel<T, LG, 4><<<n, 256, 0, stream>>>(c, r.hb, r.head_blocks, r.row_blocks, out, s);
    else attn_rows_fwd_kernel<T, LG, 0><<<n, 256, 0, stream>>>(c, r.hb, r.head_blocks, r.row_blocks, out, s);
  });
}

template <typename T, int LG, bool NT>
int bwd_by_group(const AttnArgs& a, const AttnBwd& b, T* gq, T* gk, T* gv, hipStream_t stream) {
  const RowGrid r = row_grid(a, LG);
  FMD_REQUIRE(r.blocks < (1ll << 32));
  return launch_ranges(r.blocks, [&](unsigned n, int64_t first) {
    AttnArgs c = a;
    c.block0 = (uint32_t)first;
    if (a.group == 1) attn_rows_bwd_kernel<T, LG, 1, NT><<<n, 256, 0, stream>>>(c, b, r.hb, r.head_blocks, r.row_blocks, gq, gk, gv);
    else if (a.group == 2) attn_rows_bwd_kernel<T, LG, 2, NT><<<n, 256, 0, stream>>>(c, b, r.hb, r.head_blocks, r.row_blocks, gq, gk, gv);
    else if (a.group == 4) attn_rows_bwd_kernel<T, LG, 4, NT><<<n, 256, 0, stream>>>(c, b, r.hb, r.head_blocks, r.row_blocks, gq, gk, gv);
    else attn_rows_bwd_kernel<T, LG, 0, NT><<<n, 256, 0, stream>>>(c, b, r.hb, r.head_blocks, r.row_blocks, gq, gk, gv);
  });
}

template <typename T, int LG>
int bwd(const AttnArgs& a, const AttnBwd& b, T* gq, T* gk, T* gv, hipStream_t stream) {
  const bool nt = a.tk * a.kv_heads * a.dim * 2 * (int64_t)sizeof(T) >= kStreamBytes;
  return nt ? bwd_by_group<T, LG, true>(a, b, gq, gk, gv, stream) : bwd_by_group<T, LG, false>(a, b, gq, gk, gv, stream);
}

}  // namespace

template <typename T>
int attn_rows_fwd(const AttnArgs& a, T* out, const AttnSaved& s, hipStream_t stream) {
  if (a.dim <= 8) return fwd<T, 1>(a, out, s, stream);
  if (a.dim <= 16) return fwd<T, 2>(a, out, s, stream);
  if (a.dim <= 32) return fwd<T, 4>(a, out, s, stream);
  if (a.dim <= 64) return fwd<T, 8>(a, out, s, stream);
  return fwd<T, 16>(a, out, s, stream);
}

template <typename T>
int attn_rows_bwd(const AttnArgs& a, const AttnBwd& b, T* gq, T* gk, T* gv, hipStream_t stream) {
  if (a.dim <= 8) return bwd<T, 1>(a, b, gq, gk, gv, stream);
  if (a.dim <= 16) return bwd<T, 2>(a, b, gq, gk, gv, stream);
  if (a.dim <= 32) return bwd<T, 4>(a, b, gq, gk, gv, stream);
  if (a.dim <= 64) return bwd<T, 8>(a, b, gq, gk, gv, stream);
  return bwd<T, 16>(a, b, gq, gk, gv, stream);
}

template int attn_rows_fwd<float>(const AttnArgs&, float*, const AttnSaved&, hipStream_t);
template int attn_rows_fwd<__bf16>(const AttnArgs&, __bf16*, const AttnSaved&, hipStream_t);
template int attn_rows_bwd<float>(const AttnArgs&, const AttnBwd&, float*, float*, float*, hipStream_t);
template int attn_rows_bwd<__bf16>(const AttnArgs&, const AttnBwd&, __bf16*, __bf16*, __bf16*, hipStream_t);
