// The gated feed-forward block y = h Wd^T, h = act(x Wg^T) * (x Wu^T), and its gradients.
//
// In one of three forms, by measured times (one_kernel, direct_forward, direct_backward): one kernel each way for small weights
// (ffn_block.h); products straight from memory to registers for few rows (direct_product.h); otherwise tiles in LDS (tile_product.h). The
// last two are four or five launches, each a product with what follows it as its epilogue:
//   gate, up -> h            both projections of a tile in one workgroup; the factors stay in registers and h alone is written
//   y = h Wd^T
//   gh = gy Wd -> dg, du     dg = gh u act'(g), du = gh act(g)
//   gx = dg Wg + du Wu       one product with K of two parts
//   gWg = dg^T x, gWu = du^T x, gWd = gy^T h   one launch
// The backward pass takes g and u from the forward in float32: in bf16 their rounding alone would leave dg and du two roundings off,
// and gx with them. h, dg and du are operands of the next product in two planes of bf16 (16 bits; float32: in three), so that a bf16
// result has the error of one rounding, its own. Of one plane they would cost half as many matrix instructions, with 1.41 times the error.
//
// Bound by the matrix cores from some hundred rows on, by reading the weights below. bf16, 8 192 rows of 2 048 x 5 504 (us, and the
// rate of its bf16 products, two a multiply-add for h, dg and du): projections 459 (800 TFLOP/s), y 312 (1 180; 170 with h of one plane), dg and
// du 352 (525: their epilogue moves 733 MB besides), gx 622 (1 190; 323), weights 977 (1 130; 503). float32 (six bf16 products a
// multiply-add), 16 875 rows of 256 x 680, all gradients: 577 us (92 TFLOP/s). bf16, 16 rows of 2 048 x 5 504: 32 us.
#include "ffn_block.h"

namespace {

// ---------------------------------------------------------------------------------------- operands

// A matrix [rows, cols] as the products read it: bf16, rows of `ld` elements (a multiple of 8, the rest zero), three planes of
// float32.
struct LayJob {
  const void* src;
  int64_t src_ld;
  __bf16* dst;
  int64_t rows, cols, ld, plane;
  int32_t wide;  // source rows in whole 16-byte vectors
  uint32_t first;
};

constexpr int kLayJobs = 5;
constexpr int64_t kMostBlocks = 1 << 22;

struct LayArgs {
  LayJob job[kLayJobs];
  int32_t count;
  uint32_t block0;  // first workgroup of this launch
};

template <bool F32>
__global__ void __launch_bounds__(256) ffn_lay_kernel(LayArgs a) {
  int n = 0;
#pragma unroll
  for (int i = 1; i < kLayJobs; ++i)
    if (i < a.count && a.block0 + blockIdx.x >= a.job[i].first) n = i;
  const LayJob& j = a.job[n];
  const int64_t chunks = j.ld / 8, i = (int64_t)(a.block0 + blockIdx.x - j.first) * 256 + threadIdx.x;
  if (i >= j.rows * chunks) return;
  const int64_t row = i / chunks, col = (i - row * chunks) * 8;
  const bool whole = j.wide && col + 8 <= j.cols;
  __bf16* dst = j.dst + row * j.ld + col;
  if (F32) {
    const float* src = static_cast<const float*>(j.src) + row * j.src_ld + col;
    float4 lo, hi;
    if (whole) {
      lo = reinterpret_cast<const float4*>(src)[0];
      hi = reinterpret_cast<const float4*>(src)[1];
    } else {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = col + e < j.cols ? src[e] : 0.f;
      lo = make_float4(v[0], v[1], v[2], v[3]);
      hi = make_float4(v[4], v[5], v[6], v[7]);
    }
    fmd_bf16x4 l[3], h[3];
    x3_split(lo, l[0], l[1], l[2]);
    x3_split(hi, h[0], h[1], h[2]);
#pragma unroll
    for (int p = 0; p < 3; ++p)
      *reinterpret_cast<fmd_bf16x8*>(dst + p * j.plane) = __builtin_shufflevector(l[p], h[p], 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    const __bf16* src = static_cast<const __bf16*>(j.src) + row * j.src_ld + col;
    fmd_bf16x8 v;
    if (whole) {
      v = *reinterpret_cast<const fmd_bf16x8*>(src);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = col + e < j.cols ? src[e] : (__bf16)0.f;
    }
    *reinterpret_cast<fmd_bf16x8*>(dst) = v;
  }
}

// ---------------------------------------------------------------------------------------- epilogues

__device__ __forceinline__ void put_operand(__bf16* p, int64_t plane, int planes, const float (&v)[4]) {
  if (planes == 3)
    put_planes<3>(p, plane, v);
  else
    put_planes<2>(p, plane, v);
}

// h [rows, ld] (zero in the columns past hidden), and g, u [rows, ld] for the backward pass
struct GatedEpi {
  __bf16* h;
  float *gate, *up;  // nullable
  int64_t rows, hidden, ld, plane;
  int32_t act, planes;
  typedef TpNothing Fetch;
  __device__ __forceinline__ Fetch fetch(int64_t, int64_t) const { return {}; }
  __device__ __forceinline__ void operator()(int, int64_t m, int64_t n, float4 g, float4 u, Fetch) const {
    if (m >= rows || n >= ld) return;
    const float gv[4] = {g.x, g.y, g.z, g.w}, uv[4] = {u.x, u.y, u.z, u.w};
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = n + e < hidden ? activation(gv[e], act).value * uv[e] : 0.f;
    put_operand(h + m * ld + n, plane, planes, v);
    if (gate) {
      store_stream(reinterpret_cast<float4*>(gate + m * ld + n), g);
      store_stream(reinterpret_cast<float4*>(up + m * ld + n), u);
    }
  }
};

// dg, du [2, rows, ld] from gh
struct GatedBackEpi {
  __bf16* d;
  const float *gate, *up;
  int64_t rows, hidden, ld, plane;
  int32_t act, planes;
  struct Fetch {
    float4 g, u;
  };
  __device__ __forceinline__ Fetch fetch(int64_t m, int64_t n) const {
    const int64_t at = (m < rows ? m : rows - 1) * ld + (n < ld ? n : ld - 4);
    return {*reinterpret_cast<const float4*>(gate + at), *reinterpret_cast<const float4*>(up + at)};
  }
  __device__ __forceinline__ void operator()(int, int64_t m, int64_t n, float4 gh, float4, const Fetch& f) const {
    if (m >= rows || n >= ld) return;
    const float4 g = f.g, u = f.u;
    const float hv[4] = {gh.x, gh.y, gh.z, gh.w}, gv[4] = {g.x, g.y, g.z, g.w}, uv[4] = {u.x, u.y, u.z, u.w};
    float dg[4], du[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const ActValue a = activation(gv[e], act);
      const bool in = n + e < hidden;
      dg[e] = in ? hv[e] * uv[e] * a.slope : 0.f;
      du[e] = in ? hv[e] * a.value : 0.f;
    }
    put_operand(d + m * ld + n, plane, planes, dg);
    put_operand(d + (rows + m) * ld + n, plane, planes, du);
  }
};

// results [rows_m, rows_n] of each problem, in the features' type
struct StoreEpi {
  void* out[kTpProblems];
  int64_t rows_m[kTpProblems], rows_n[kTpProblems];
  int32_t bf16;
  typedef TpNothing Fetch;
  __device__ __forceinline__ Fetch fetch(int64_t, int64_t) const { return {}; }
  __device__ __forceinline__ void operator()(int i, int64_t m, int64_t n, float4 v, float4, Fetch) const {
    const int64_t width = i == 0 ? rows_n[0] : i == 1 ? rows_n[1] : rows_n[2];
    if (m >= (i == 0 ? rows_m[0] : i == 1 ? rows_m[1] : rows_m[2]) || n >= width) return;
    void* o = i == 0 ? out[0] : i == 1 ? out[1] : out[2];
    const float e[4] = {v.x, v.y, v.z, v.w};
    if (bf16) {
      __bf16* p = static_cast<__bf16*>(o) + m * width + n;
      if (width % 4 == 0) {
        fmd_bf16x4 x;
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = (__bf16)e[k];
        *reinterpret_cast<fmd_bf16x4*>(p) = x;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (n + k < width) p[k] = (__bf16)e[k];
      }
    } else {
      float* p = static_cast<float*>(o) + m * width + n;
      if (width % 4 == 0) {
        *reinterpret_cast<float4*>(p) = v;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (n + k < width) p[k] = e[k];
      }
    }
  }
};

// ---------------------------------------------------------------------------------------- host

template <bool NA, bool MA, bool GATED>
struct Shapes {
  typedef TpShape<TpBf16, 2, 4, 4, 2, NA, MA, GATED, 2> Large;   // 256 x 256, 8 waves, one workgroup a CU
  typedef TpShape<TpBf16, 2, 2, 2, 2, NA, MA, GATED, 2> Middle;  // 128 x 128, 4 waves, two
  typedef TpShape<TpBf16, 1, 2, 2, 1, NA, MA, GATED, 2> Small;   // 64 x 64, 2 waves
};

template <typename S>
int64_t count_tiles(TpArgs& a) {
  int64_t tiles = 0;
  for (int i = 0; i < a.count; ++i) tiles = tp_tiles<S>(a.p[i], tiles);
  return tiles;
}

// The tile and the split of K with the least time (tp_plan).
template <typename Sh, typename Fn>
int with_shape(TpArgs& a, float heavy, const Fn& fn) {
  int64_t slices = 0;
  for (int i = 0; i < a.count; ++i) {
    const int64_t s = fmd_cdiv(2 * a.p[i].k, kTpSlice) * a.p[i].parts * a.p[i].pairs.count;
    slices = i == 0 || s < slices ? s : slices;
  }
  int64_t tiles = count_tiles<typename Sh::Large>(a);
  if (tiles > kTpMostTiles) return FMD_EINVAL;
  const TpPlan large = tp_plan<typename Sh::Large>(tiles, slices, heavy);
  if (tiles >= 1024) return fn(typename Sh::Large{}, large);
  const TpPlan middle = tp_plan<typename Sh::Middle>(count_tiles<typename Sh::Middle>(a), slices, heavy);
  const TpPlan small = tp_plan<typename Sh::Small>(count_tiles<typename Sh::Small>(a), slices, heavy);
  if (small.time < middle.time && small.time < large.time) return fn(typename Sh::Small{}, small);
  if (middle.time < large.time) {
    count_tiles<typename Sh::Middle>(a);
    return fn(typename Sh::Middle{}, middle);
  }
  count_tiles<typename Sh::Large>(a);
  return fn(typename Sh::Large{}, large);
}

int64_t up8(int64_t x) { return (x + 7) & ~int64_t(7); }
int64_t up256(int64_t x) { return (x + 255) & ~int64_t(255); }

// Everything that a call lays out in its workspace; with a null base the sizes alone.
struct Space {
  char* base;
  int64_t used = 0;
  template <typename T = void>
  T* take(int64_t bytes) {
    T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += up256(bytes);
    return p;
  }
};

struct Ffn {
  int32_t bf16, act, lay;  // lay: bits of the operands that are laid out in the workspace: x, gate and up, down, gy
  int64_t rows, width, hidden, out;
  int64_t hp() const { return up8(hidden); }
  int planes() const { return bf16 ? 1 : 3; }  // of x, gy and the weights
  int kept() const { return bf16 ? 2 : 3; }    // of h, dg and du
  TpPairs pairs() const { return bf16 ? kTpPlain : kTpThree; }
  TpPairs kept_m() const { return bf16 ? kTpTwoM : kTpThree; }
  TpPairs kept_n() const { return bf16 ? kTpTwoN : kTpThree; }
};

// an operand: the caller's matrix, or its layout in the workspace
struct Matrix {
  const void* p;
  int64_t ld, plane;
};

struct Layer {
  LayArgs args{};
  int64_t blocks = 0;
  Matrix add(const Ffn& f, Space& s, bool lay, const void* src, int64_t ld, int64_t rows, int64_t cols) {
    if (!lay) return {src, ld, 0};
    const int64_t wide = up8(cols);
    __bf16* dst = s.take<__bf16>(rows * wide * 2 * f.planes());
    LayJob& j = args.job[args.count++];
    const int size = f.bf16 ? 2 : 4;
    j = {src, ld, dst, rows, cols, wide, rows * wide,
         (int32_t)(ld * size % 16 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0), (uint32_t)blocks};
    blocks += fmd_cdiv(rows * wide / 8, 256);
    return {dst, wide, rows * wide};
  }
  int launch(const Ffn& f, hipStream_t stream) {
    FMD_REQUIRE(blocks < (int64_t(1) << 32));
    for (int64_t first = 0; first < blocks; first += kMostBlocks) {  // a launch takes fewer than 2^32 threads
      const unsigned n = (unsigned)(blocks - first < kMostBlocks ? blocks - first : kMostBlocks);
      args.block0 = (uint32_t)first;
      if (f.bf16)
        ffn_lay_kernel<false><<<n, 256, 0, stream>>>(args);
      else
        ffn_lay_kernel<true><<<n, 256, 0, stream>>>(args);
      FMD_CHECK_LAUNCH();
    }
    return FMD_OK;
  }
};

TpOperand operand(const Matrix& a, const Matrix& b) { return tp_operand(a.p, b.p, a.ld, a.plane, 2); }

bool direct(const void* p, int64_t ld, int64_t cols) {
  return ld % 8 == 0 && cols % 8 == 0 && ld * 2 <= kTpMostLd && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

// A launch of one kind of product: its partial sums' size, or the launch itself
template <typename Sh, typename Epi>
int product(TpArgs& a, Space& s, bool run, const Epi& epi, hipStream_t stream) {
  return with_shape<Sh>(a, sizeof(typename Epi::Fetch) > 16 ? 3.f : 1.f, [&](auto shape, const TpPlan& plan) {
    typedef decltype(shape) S;
    const int64_t before = s.used;
    void* partial = s.take(plan.partial);
    const int status = run ? tp_launch<S>(a, plan, partial, epi, stream) : FMD_OK;
    s.used = before;  // the next product's sums take the same place
    a.partial = nullptr;
    if (!run) s.used += up256(plan.partial);  // sizes: the caller keeps the largest
    return status;
  });
}

TpArgs one(const TpOperand& n, const TpOperand& m, int64_t rows_n, int64_t rows_m, int64_t k, int parts, const TpPairs& pairs) {
  TpArgs a{};
  a.p[0] = {n, m, rows_n, rows_m, k, parts, pairs, 0, 0, 0};
  a.count = 1;
  return a;
}

struct Forward {
  const void *x, *gate, *up, *down;
  int64_t x_ld, gate_ld, down_ld;  // gate_ld: of both projections
  void* y;
  float* saved;    // g, u [2, rows, hp], or null
  __bf16* hidden;  // [planes, rows, hp], or null: in the workspace
};

// Whether the products of a pass go straight from memory to registers (direct_product.h) or through tiles in LDS: by the multiply-adds
// of the forward pass and the rows, where the two forms' times meet. us of tiles, straight:
// float32, forward: 1 000 rows of 256 x 680 42 39, 2 000 47 53; 200 of 512 x 1 376 47 40, 500 53 58; 200 of 768 x 2 048 59 54, 400 73 93; 4 000 of
//   128 x 344 37 33; 10 000 of 64 x 256 36 39, of 96 x 192 38 41; 64 of 2 048 x 5 504 157 120; 16 of 4 096 x 11 008 538 153.
// float32, VJP for x: 500 of 256 x 680 44 26, 1 000 46 57; 64 of 512 x 1 376 44 40, 130 47 45, 200 48 53 (but 500 67 61); 32 of 1 024 x 2 736 60 50, 64
//   62 75; 2 000 of 128 x 344 39 37, 4 000 44 45; 32 of 2 048 x 5 504 153 105, 64 158 169; 16 of 4 096 x 11 008 530 224.
// bf16, forward: 500 of 256 x 680 21.8 14.3, 1 000 23.4 25.5; 1 000 of 128 x 344 16.5 13.0, 2 000 17.7 19.4; 130 of 512 x 1 376 20.6 19.7, 200 21.4
//   24.8; 32 of 1 024 x 2 736 22.8 20.0, 64 25.8 29.3; 64 of 768 x 2 048 22.2 27.7; 16 of 2 048 x 5 504 38.5 34.4, 32 40.2 45.7; 16 of 4 096 x 11 008
//   92.7 82.1.
// bf16, VJP for x: 300 of 256 x 680 23.6 23.9, 500 26.3 18.8, 1 000 31.3 39.9; 1 000 of 128 x 344 21.5 19.3, 2 000 27.2 30.1; 32 of 512 x 1 376 26.9
//   21.7, 64 27.7 28.4, 130 30.3 38.0; 16 of 768 x 2 048 26.3 25.6, of 1 024 x 2 736 33.1 32.5, of 2 048 x 5 504 40.6 61.6 (weights are read across
//   their rows, two bytes a lane).
bool direct_forward(const Ffn& f) {
  const double work = (double)f.rows * f.hidden * (2 * f.width + f.out);
  if (f.bf16) return f.rows <= 16 || work <= (f.rows <= 512 ? 2.7e8 : 2e8);
  return f.rows <= 64 || work <= (f.rows <= 4096 ? 9.5e8 : 2.4e8);
}
bool direct_backward(const Ffn& f) {
  const double weights = (double)f.hidden * (2 * f.width + f.out), work = weights * f.rows;
  if (f.bf16) return weights <= 2.2e6 && work <= (weights <= 6e5 && f.rows <= 512 ? 2.7e8 : 1.33e8);
  return f.rows <= 32 || work <= 3e8;
}

// Whether the whole block is one kernel: its hidden layer (in the backward pass the two gradients of it) fits LDS for 16 rows, and the
// weights, which every workgroup walks through, are few. us of the forward pass and of the VJP for x, the better of the other forms and in one
// kernel: 64 x 128 float32, 135 rows 10.6 10.5, 10.9 13.5, 1 000 rows 10.7 8.8, 12.4 13.6, 10 000 rows 24.7 18.5, 36.2 29.5; bf16 8.2 6.7, 11.4 10.2;
// 10.8 5.9, 12.3 10.3; 14.0 10.9, 20.8 19.7. 64 x 256 float32, 135 rows 9.7 12.7, 11.6 23.3, 10 000 rows 35.8 30.3, 42.8 52.2; bf16 8.8 8.0, 11.7 16.9 and
// 19.5 16.7, 28.1 34.9.
bool one_kernel(const Ffn& f) {
  const int64_t weights = f.hidden * (2 * f.width + f.out);
  return weights <= (!f.bf16 && f.rows >= 4096 ? 50000 : 25000) && block_lds((int)f.hidden, f.kept(), 16, true) <= kBlockLds;
}

template <typename T, bool BACK>
int block(const Ffn& f, FfnBlock a, hipStream_t stream) {
  const auto launch = [&](auto mt) {
    constexpr int MT = decltype(mt)::value;
    for (a.row0 = 0; a.row0 < f.rows; a.row0 += kMostBlocks * 16 * MT) {
      const int64_t left = fmd_cdiv(f.rows - a.row0, 16 * MT);
      ffn_block_kernel<T, MT, BACK><<<(unsigned)(left < kMostBlocks ? left : kMostBlocks), kBlockThreads,
                                      block_lds((int)f.hidden, f.kept(), 16 * MT, BACK), stream>>>(a);
      FMD_CHECK_LAUNCH();
    }
    return (int)FMD_OK;
  };
  // 32 rows of a workgroup where those fill the card
  if (f.rows >= 32 * kTpCus && block_lds((int)f.hidden, f.kept(), 32, BACK) <= kBlockLds) return launch(std::integral_constant<int, 2>{});
  return launch(std::integral_constant<int, 1>{});
}

int32_t wide_rows(const Ffn& f, const void* p, int64_t ld, int64_t k) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * (f.bf16 ? 2 : 4) % 16 == 0 && k % 8 == 0;
}

DpOperand in_memory(const Ffn& f, const void* a, const void* b, int64_t ld, int64_t k) {
  return {{a, b}, ld, 0, wide_rows(f, a, ld, k) && wide_rows(f, b, ld, k)};
}
DpOperand planes_in_memory(const Ffn& f, const __bf16* a, const __bf16* b, int64_t plane) { return {{a, b}, f.hp(), plane, 1}; }

template <bool N_ACROSS, bool GATED, bool OWN, typename Epi>
int straight(const Ffn& f, const DpArgs& a, const Epi& epi, hipStream_t stream) {  // OWN: m is h, dg or du
  if (f.bf16) return dp_product<__bf16, N_ACROSS, GATED, OWN>(a, epi, stream);
  return dp_product<float, N_ACROSS, GATED, OWN>(a, epi, stream);
}

FfnBlock block_args(const Ffn& f, const Forward& io, const void* gy, int64_t gy_ld, void* result) {
  return {io.x, io.gate, io.up, io.down, gy, io.x_ld, io.gate_ld, io.down_ld, gy_ld, wide_rows(f, io.x, io.x_ld, f.width),
          wide_rows(f, io.gate, io.gate_ld, f.width) && wide_rows(f, io.up, io.gate_ld, f.width), wide_rows(f, io.down, io.down_ld, f.hidden),
          wide_rows(f, gy, gy_ld, f.out), f.rows, (int32_t)f.width, (int32_t)f.hidden, (int32_t)f.out, f.act, result, nullptr, nullptr, f.hp(), 0};
}

int forward(const Ffn& f, const Forward& io, Space& s, bool run, hipStream_t stream, int64_t* size) {
  const int64_t hp = f.hp(), plane = f.rows * hp;
  const StoreEpi store{{io.y}, {f.rows}, {f.out}, f.bf16};
  if (one_kernel(f)) {
    if (size) *size = 0;
    if (!run) return FMD_OK;
    const FfnBlock a = block_args(f, io, nullptr, 0, io.y);
    return f.bf16 ? block<__bf16, false>(f, a, stream) : block<float, false>(f, a, stream);
  }
  if (direct_forward(f)) {
    __bf16* h = io.hidden ? io.hidden : s.take<__bf16>(plane * 2 * f.kept());
    if (size) *size = s.used;
    if (!run) return FMD_OK;
    const GatedEpi gated{h, io.saved, io.saved ? io.saved + plane : nullptr, f.rows, f.hidden, hp, plane, f.act, f.kept()};
    DpOperand weights = in_memory(f, io.gate, io.up, io.gate_ld, f.width);
    const DpArgs first{weights, in_memory(f, io.x, io.x, io.x_ld, f.width), f.hidden, f.rows, f.width, 1, 0, 0};
    int status = straight<false, true, false>(f, first, gated, stream);
    if (status) return status;
    const DpArgs second{in_memory(f, io.down, io.down, io.down_ld, f.hidden), planes_in_memory(f, h, h, plane), f.out, f.rows, f.hidden, 1, 0, 0};
    return straight<false, false, true>(f, second, store, stream);
  }
  Layer lay;
  const Matrix x = lay.add(f, s, f.lay & 1, io.x, io.x_ld, f.rows, f.width);
  const Matrix g = lay.add(f, s, f.lay & 2, io.gate, io.gate_ld, f.hidden, f.width);
  const Matrix u = lay.add(f, s, f.lay & 2, io.up, io.gate_ld, f.hidden, f.width);
  const Matrix d = lay.add(f, s, f.lay & 4, io.down, io.down_ld, f.out, f.hidden);
  __bf16* h = io.hidden ? io.hidden : s.take<__bf16>(plane * 2 * f.kept());
  if (run) {
    const int status = lay.launch(f, stream);
    if (status) return status;
  }
  int64_t most = s.used;
  const int64_t base = s.used;
  TpArgs a = one(operand(g, u), operand(x, x), f.hidden, f.rows, f.width, 1, f.pairs());
  const GatedEpi gated{h, io.saved, io.saved ? io.saved + plane : nullptr, f.rows, f.hidden, hp, plane, f.act, f.kept()};
  int status = product<Shapes<false, false, true>>(a, s, run, gated, stream);
  if (status) return status;
  most = s.used > most ? s.used : most;
  s.used = base;
  const Matrix hm{h, hp, plane};
  a = one(operand(d, d), operand(hm, hm), f.out, f.rows, f.hidden, 1, f.kept_m());
  status = product<Shapes<false, false, false>>(a, s, run, store, stream);
  if (status) return status;
  most = s.used > most ? s.used : most;
  if (size) *size = most;
  return FMD_OK;
}

struct Backward {
  Forward in;
  const void* gy;
  int64_t gy_ld;
  void *gx, *g_gate, *g_up, *g_down;  // gx, or the three weights', nullable
};

int backward(const Ffn& f, const Backward& io, bool want_x, bool want_w, Space& s, bool run, hipStream_t stream, int64_t* size) {
  const bool together = one_kernel(f), straight_on = together || direct_backward(f);
  Layer lay;
  Matrix x{}, g{}, u{}, d{}, gy{};
  if (want_w) x = lay.add(f, s, f.lay & 1, io.in.x, io.in.x_ld, f.rows, f.width);
  if (want_x && !straight_on) {
    g = lay.add(f, s, f.lay & 2, io.in.gate, io.in.gate_ld, f.hidden, f.width);
    u = lay.add(f, s, f.lay & 2, io.in.up, io.in.gate_ld, f.hidden, f.width);
  }
  if (!straight_on) d = lay.add(f, s, f.lay & 4, io.in.down, io.in.down_ld, f.out, f.hidden);
  if (want_w || !straight_on) gy = lay.add(f, s, f.lay & 8, io.gy, io.gy_ld, f.rows, f.out);
  const int64_t hp = f.hp(), plane = f.rows * hp;
  __bf16* dgu = together && !want_w ? nullptr : s.take<__bf16>(2 * plane * 2 * f.kept());
  if (run) {
    const int status = lay.launch(f, stream);
    if (status) return status;
  }
  int64_t most = s.used;
  __bf16* h = io.in.hidden;
  TpArgs a{};
  if (together) {
    h = want_w ? s.take<__bf16>(plane * 2 * f.kept()) : nullptr;
    most = s.used;
    if (run) {
      FfnBlock b = block_args(f, io.in, io.gy, io.gy_ld, io.gx);
      b.h = h;
      b.d = want_w ? dgu : nullptr;
      const int status = f.bf16 ? block<__bf16, true>(f, b, stream) : block<float, true>(f, b, stream);
      if (status) return status;
    }
  }
  const int64_t base = s.used;
  const GatedBackEpi back{dgu, io.in.saved, io.in.saved ? io.in.saved + plane : nullptr, f.rows, f.hidden, hp, 2 * plane, f.act, f.kept()};
  int status = FMD_OK;
  if (together) {
  } else if (!straight_on) {
    a = one(operand(d, d), operand(gy, gy), f.hidden, f.rows, f.out, 1, f.pairs());
    status = product<Shapes<true, false, false>>(a, s, run, back, stream);
    most = s.used > most ? s.used : most;
  } else if (run) {
    const DpArgs first{in_memory(f, io.in.down, io.in.down, io.in.down_ld, f.out), in_memory(f, io.gy, io.gy, io.gy_ld, f.out), f.hidden, f.rows, f.out, 1, 0, 0};
    status = straight<true, false, false>(f, first, back, stream);
  }
  if (status) return status;
  const Matrix dg{dgu, hp, 2 * plane}, du{dgu + plane, hp, 2 * plane};
  if (want_x && !together) {
    s.used = base;
    const StoreEpi store{{io.gx}, {f.rows}, {f.width}, f.bf16};
    if (!straight_on) {
      a = one(operand(g, u), operand(dg, du), f.width, f.rows, f.hidden, 2, f.kept_m());
      status = product<Shapes<true, false, false>>(a, s, run, store, stream);
      most = s.used > most ? s.used : most;
    } else if (run) {
      const DpArgs second{in_memory(f, io.in.gate, io.in.up, io.in.gate_ld, f.hidden), planes_in_memory(f, dgu, dgu + plane, 2 * plane), f.width, f.rows, f.hidden, 2, 0, 0};
      status = straight<true, false, true>(f, second, store, stream);
    }
    if (status) return status;
  }
  if (want_w) {
    s.used = base;
    const Matrix hm{h, hp, plane};
    a = one(operand(x, x), operand(dg, dg), f.width, f.hidden, f.rows, 1, f.kept_m());
    a.p[1] = {operand(x, x), operand(du, du), f.width, f.hidden, f.rows, 1, f.kept_m(), 0, 0, 0};
    a.p[2] = {operand(hm, hm), operand(gy, gy), f.hidden, f.out, f.rows, 1, f.kept_n(), 0, 0, 0};
    a.count = 3;
    const StoreEpi store{{io.g_gate, io.g_up, io.g_down}, {f.hidden, f.hidden, f.out}, {f.width, f.width, f.hidden}, f.bf16};
    status = product<Shapes<true, true, false>>(a, s, run, store, stream);
    if (status) return status;
    most = s.used > most ? s.used : most;
  }
  if (size) *size = most;
  return FMD_OK;
}

bool sizes_fit(const Ffn& f) {
  return f.rows >= 1 && f.width >= 1 && f.hidden >= 1 && f.out >= 1 && f.rows < (int64_t(1) << 31) &&
         (f.bf16 || f.lay == 15) && up8(f.width) * 2 <= kTpMostLd && up8(f.hidden) * 2 <= kTpMostLd && up8(f.out) * 2 <= kTpMostLd &&
         f.act >= kActNone && f.act <= kActRelu;
}

bool layouts_fit(const Ffn& f, const Forward& io) {
  if (!f.bf16) return true;
  return ((f.lay & 1) || direct(io.x, io.x_ld, f.width)) &&
         ((f.lay & 2) || (direct(io.gate, io.gate_ld, f.width) && direct(io.up, io.gate_ld, f.width))) &&
         ((f.lay & 4) || direct(io.down, io.down_ld, f.hidden));
}

}  // namespace

extern "C" {

int32_t fmd_gated_ffn_saves(int32_t bf16, int64_t rows, int64_t width, int64_t hidden, int64_t out) {
  const Ffn f{bf16, 0, 15, rows, width, hidden, out};
  return sizes_fit(f) && !one_kernel(f);
}

int64_t fmd_gated_ffn_work_size(int32_t bf16, int64_t rows, int64_t width, int64_t hidden, int64_t out, int32_t lay,
                                int32_t keep_hidden) {
  const Ffn f{bf16, 0, lay, rows, width, hidden, out};
  if (!sizes_fit(f)) return 0;
  Space s{nullptr};
  Forward io{};
  io.hidden = keep_hidden ? reinterpret_cast<__bf16*>(16) : nullptr;
  int64_t size = 0;
  forward(f, io, s, false, nullptr, &size);
  return size;
}

int fmd_gated_ffn(int32_t bf16, int32_t act, int32_t lay, const void* x, int64_t x_ld, const void* gate,
                  const void* up, int64_t gate_ld, const void* down, int64_t down_ld, int64_t rows, int64_t width, int64_t hidden,
                  int64_t out, void* y, float* saved, void* hidden_out, void* work, hipStream_t stream) {
  const Ffn f{bf16, act, lay, rows, width, hidden, out};
  const Forward io{x, gate, up, down, x_ld, gate_ld, down_ld, y, saved, static_cast<__bf16*>(hidden_out)};
  FMD_REQUIRE(sizes_fit(f) && layouts_fit(f, io) && x && gate && up && down && y);
  int64_t size = 0;
  Space none{nullptr}, s{static_cast<char*>(work)};
  const int status = forward(f, io, none, false, nullptr, &size);
  if (status) return status;  // before anything is laid out
  FMD_REQUIRE(work || !size);
  return forward(f, io, s, true, stream, nullptr);
}

int64_t fmd_gated_ffn_bwd_work_size(int32_t bf16, int64_t rows, int64_t width, int64_t hidden, int64_t out, int32_t lay,
                                    int32_t want_x, int32_t want_w) {
  const Ffn f{bf16, 0, lay, rows, width, hidden, out};
  if (!sizes_fit(f)) return 0;
  Space s{nullptr};
  const Backward io{};
  int64_t size = 0;
  backward(f, io, want_x, want_w, s, false, nullptr, &size);
  return size;
}

int fmd_gated_ffn_bwd(int32_t bf16, int32_t act, int32_t lay, const void* x, int64_t x_ld, const void* gate,
                      const void* up, int64_t gate_ld, const void* down, int64_t down_ld, int64_t rows, int64_t width,
                      int64_t hidden, int64_t out, const void* gy, int64_t gy_ld, const float* saved, const void* hidden_in,
                      void* gx, void* g_gate, void* g_up, void* g_down, void* work, hipStream_t stream) {
  const Ffn f{bf16, act, lay, rows, width, hidden, out};
  Backward io{};
  io.in = {x, gate, up, down, x_ld, gate_ld, down_ld, nullptr, const_cast<float*>(saved),
           static_cast<__bf16*>(const_cast<void*>(hidden_in))};
  io.gy = gy;
  io.gy_ld = gy_ld;
  io.gx = gx;
  io.g_gate = g_gate;
  io.g_up = g_up;
  io.g_down = g_down;
  FMD_REQUIRE(sizes_fit(f) && layouts_fit(f, io.in) && x && gate && up && down && gy && (saved || one_kernel(f)));
  FMD_REQUIRE(!bf16 || (lay & 8) || direct(gy, gy_ld, out));
  FMD_REQUIRE(!g_gate || (g_up && g_down && (hidden_in || one_kernel(f))));
  int64_t size = 0;
  Space none{nullptr}, s{static_cast<char*>(work)};
  const int status = backward(f, io, gx != nullptr, g_gate != nullptr, none, false, nullptr, &size);
  if (status) return status;
  FMD_REQUIRE(work || !size);
  return backward(f, io, gx != nullptr, g_gate != nullptr, s, true, stream, nullptr);
}

}  // extern "C"
