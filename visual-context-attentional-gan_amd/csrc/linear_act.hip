// Linear layers with bias, activation and residual in the product's epilogue, forward and gradients, on fp32 and 16-bit
// tensors of any size, row stride and alignment:
//
//   z = x W^T + b     y = act(z) + r          (one pass over the product; training keeps z, see ZOf)
//   dz = gy act'(z)   db = sum_m dz           (one pass over gy and z)
//   dx = dz W         dW = dz^T x             (products with one or both operands read along their columns)
//
// All three products are C[m][n] = sum_k A(m, k) B(n, k); an operand is stored either with k contiguous (x, W in the
// forward pass, dz in dx) or with its own index contiguous (W in dx, dz and x in dW).  Neither is ever transposed in
// memory: a column-major operand is staged as it lies and transposed on the way from LDS to the registers.
//
// Arithmetic: 16-bit tensors of the library's element type take one product with fp32 accumulation.  fp32 tensors take
// the exact fp32 MFMA (nsplit 0) or are split in registers into 16-bit parts (nsplit 3: hi hi + hi lo + lo hi; 1: hi).
// Bias, activation and residual are applied to the fp32 accumulator, so a result is rounded once.
#include <initializer_list>
#include <type_traits>

#include "common.h"

namespace {

enum { MODE_16 = 0, MODE_F32 = 1, MODE_S3 = 2, MODE_S1 = 3 };   // 16-bit tensors; fp32: exact, three products, one

template <int MODE> struct ElemOf { typedef float T; };
template <> struct ElemOf<MODE_16> { typedef vca_e16 T; };

// What the value under the activation is kept in for the backward pass.  Its rounding enters dz next to dz's own, so
// it has to be the smaller of the two: three more bits than bf16 in the same room, fp32 beside half.  Half's range is
// narrower than bf16's at both ends.  At the upper one the slopes are 0, 1 or flat, an infinity included.  At the
// lower one the smooth slopes are flat too, but the kinked ones turn on the sign, so a positive value stays positive
// (keep_z).
#ifdef VCA_E16_FP16
typedef float vca_z16;
#else
typedef _Float16 vca_z16;
#endif
template <typename T> struct ZOf { typedef float type; };
template <> struct ZOf<vca_e16> { typedef vca_z16 type; };

typedef short s16x4 __attribute__((ext_vector_type(4)));

struct MatArgs {
  const void *a, *b, *bias, *res;
  void *c, *z;
  float* part;                        // [ksplit][M][npad] partial products (ksplit > 1)
  long long lda, ldb, ldc, ldr;       // elements
  int M, N, K;
  int ntm, ntn, ksplit, cpz, npad;    // tiles, reduction ranges, chunks a range, padded columns of a partial product
  int act;
  float slope;
};

// 16 bytes from any address that is aligned to its element: gfx950 takes unaligned wide accesses, the packed type makes
// the compiler use them.
struct __attribute__((packed, aligned(2))) Any16 { uint4 u; };

template <typename T> union Vec16 {
  uint4 u;
  T e[16 / sizeof(T)];
};

// ------------------------------------------------------------------------------------------------
// activations, in fp32
//
// FULL, for fp32 tensors: the exponential is the library's, and gelu carries along what its argument's square loses, so
// that value and slope are good to some 20 half ulps of their terms (the tanh form of gelu: and 6 of its exponent).
// 16-bit tensors, whose own rounding is 2^13 of those and more, take the hardware's exponential: an argument k costs it
// some |k| half ulps.  (fp32 4800 x 512 -> 1280 with gelu, forward and all gradients: 209 us, 205 with the hardware's.)
// ------------------------------------------------------------------------------------------------
constexpr float GELU_C = 0.7978845608028654f, GELU_A = 0.044715f;   // sqrt(2 / pi)

__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// s = 1 / (1 + e^-x) and its slope d = s (1 - s); 0 and 1 at the ends
template <bool FULL>
__device__ __forceinline__ float sigmoid_f(float x, float& d) {
  if (FULL) {                                              // from e^-|x|: no overflow, and no difference in d
    const float e = expf(-fabsf(x)), r = __builtin_amdgcn_rcpf(1.f + e);
    d = e * r * r;
    return x < 0.f ? e * r : r;
  }
  const float s = __builtin_amdgcn_rcpf(1.f + fast_exp(-x));
  d = s * (1.f - s);
  return s;
}

// e = exp(-z^2 / 2) and Phi(-|z|), the normal distribution's tail, as t P(t) e with t = 1 / (1 + c |z|).  P and c were
// fitted for this file, for the relative error wherever the tail lies: least squares on 6000 Chebyshev nodes of t,
// reweighted until the error is level over |z| <= 15, behind which the tail is below fp32.  Degree 8 is within 3.2e-8 (12
// half ulps as evaluated) and degree 6, for 16-bit tensors, within 1.1e-6; two terms more cost 8192 x 4096 -> 4096 4 us,
// forward and backward.  So gelu keeps its digits far out on the negative side, for about half of erff's instructions.
template <bool FULL>
__device__ __forceinline__ float normal_tail(float z, float& e) {
  float a = fabsf(z), t, p;
  if (FULL) {
    a = a > 15.f ? 15.f : a;                               // (keeps infinity from the difference; a NaN stays one)
    const float h = a * a;
    e = expf(-0.5f * h);
    e -= e * (0.5f * fmaf(a, a, -h));                      // what the square lost
    t = __builtin_amdgcn_rcpf(1.f + 0.26f * a);
    p = 0.029960118f;
    p = p * t - 0.15018713f;
    p = p * t + 0.2460446f;
    p = p * t - 0.1447271f;
    p = p * t + 0.15665133f;
    p = p * t + 0.052859996f;
    p = p * t + 0.10256f;
    p = p * t + 0.10308303f;
    p = p * t + 0.10375513f;
  } else {
    e = __builtin_amdgcn_exp2f(a * a * -0.72134752f);      // log2(e) / 2
    t = __builtin_amdgcn_rcpf(1.f + 0.36f * a);
    p = 0.046522163f;
    p = p * t - 0.17793439f;
    p = p * t + 0.1784647f;
    p = p * t + 0.028258404f;
    p = p * t + 0.13909869f;
    p = p * t + 0.14188473f;
    p = p * t + 0.14370519f;
  }
  return t * p * e;
}

template <bool FULL>
__device__ __forceinline__ float act_f(float z, int act, float slope) {
  float e;
  switch (act) {
    case VCA_ACT_LEAKY: return z > 0.f ? z : z * slope;
    case VCA_ACT_RELU: return z <= 0.f ? 0.f : z;            // a NaN stays one
    case VCA_ACT_TANH: return tanhf(z);
    case VCA_ACT_GELU: {                                     // z Phi(z); the small tail is multiplied, never subtracted
      const float q = normal_tail<FULL>(z, e);
      return z * (z > 0.f ? 1.f - q : q);
    }
    case VCA_ACT_GELU_TANH: return z * sigmoid_f<FULL>(2.f * GELU_C * (z + GELU_A * z * z * z), e);   // (1 + tanh u) / 2
    case VCA_ACT_SILU: return z * sigmoid_f<FULL>(z, e);
    default: return z;
  }
}

template <bool FULL, int V>
__device__ __forceinline__ void act_all(float (&v)[V], int act, float slope) {
  switch (act) {                       // one test for the V values
#define VCA_EACH(code)                                       \
  case code: {                                               \
    _Pragma("unroll") for (int r = 0; r < V; ++r) v[r] = act_f<FULL>(v[r], code, slope); \
    break;                                                   \
  }
    VCA_EACH(VCA_ACT_LEAKY)
    VCA_EACH(VCA_ACT_RELU)
    VCA_EACH(VCA_ACT_TANH)
    VCA_EACH(VCA_ACT_GELU)
    VCA_EACH(VCA_ACT_GELU_TANH)
    VCA_EACH(VCA_ACT_SILU)
#undef VCA_EACH
    default: break;
  }
}

template <bool FULL>
__device__ __forceinline__ float act_slope(float z, int act, float slope) {
  // beyond +-200 the smooth activations' slopes are 0 or 1 to fp32's last subnormal; the clamp keeps 0 x infinity out
  // of them.  At a NaN they are one (it comes through the unclamped term), relu's is 1 and leaky's its slope, as
  // torch's are.
  const float c = fminf(fmaxf(z, -200.f), 200.f);
  float e;
  switch (act) {
    case VCA_ACT_LEAKY: return z > 0.f ? 1.f : slope;
    case VCA_ACT_RELU: return z <= 0.f ? 0.f : 1.f;
    case VCA_ACT_TANH: {
      const float h = tanhf(z);
      return 1.f - h * h;
    }
    case VCA_ACT_GELU: {
      const float q = normal_tail<FULL>(z, e);
      return (z > 0.f ? 1.f - q : q) + c * e * 0.3989422804014327f;
    }
    case VCA_ACT_GELU_TANH: {
      const float s = sigmoid_f<FULL>(2.f * GELU_C * (z + GELU_A * z * z * z), e);
      return s + c * e * 2.f * GELU_C * (1.f + 3.f * GELU_A * c * c);
    }
    case VCA_ACT_SILU: {
      const float s = sigmoid_f<FULL>(z, e);
      return s + c * e;
    }
    default: return 1.f;
  }
}

// V neighbouring elements from any address (a vector, not an array: the compiler keeps that in registers)
template <typename T, int V> struct AnyVec {
  typedef T Vec __attribute__((ext_vector_type(V)));
  Vec e;
  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(&e, p, sizeof(e)); }
};

template <typename T, int V>
__device__ __forceinline__ AnyVec<T, V> load_any(const T* p, int left) {      // left: columns that exist
  AnyVec<T, V> q;
  if (left >= V) {
    q.load(p);
  } else {
#pragma unroll
    for (int r = 0; r < V; ++r) q.e[r] = r < left ? p[r] : (T)0.f;
  }
  return q;
}

template <typename T, int V>
__device__ __forceinline__ void store_any(T* p, int left, const float (&v)[V]) {
  if (left >= V) {
    AnyVec<T, V> q;
#pragma unroll
    for (int r = 0; r < V; ++r) q.e[r] = (T)v[r];
    __builtin_memcpy(p, &q.e, sizeof(q.e));
  } else {
#pragma unroll
    for (int r = 0; r < V; ++r)
      if (r < left) p[r] = (T)v[r];
  }
}

// (a missing bias or residual takes no part in this: the branch is the same for the whole launch)
template <typename T, int V>
__device__ __forceinline__ AnyVec<T, V> bias_of(const MatArgs& g, int n) {
  AnyVec<T, V> q = {};
  if (g.bias) q = load_any<T, V>(reinterpret_cast<const T*>(g.bias) + n, g.N - n);
  return q;
}

template <typename T, int V>
__device__ __forceinline__ AnyVec<T, V> res_of(const MatArgs& g, int m, int n) {
  AnyVec<T, V> q = {};
  if (g.res) q = load_any<T, V>(reinterpret_cast<const T*>(g.res) + (size_t)m * g.ldr + n, g.N - n);
  return q;
}

// The V values under the activation as they are kept: where relu or leaky will read no more than their sign out of half
// (see ZOf), a positive one is at least half's smallest, which rounding to nearest would take to zero up to 2^-25.
template <typename Z, int V>
__device__ __forceinline__ void keep_z(const MatArgs& g, int m, int n, const float (&v)[V]) {
  Z* p = reinterpret_cast<Z*>(g.z) + (size_t)m * g.N + n;
  if (sizeof(Z) == 2 && (g.act == VCA_ACT_RELU || g.act == VCA_ACT_LEAKY)) {
    float k[V];
#pragma unroll
    for (int r = 0; r < V; ++r) k[r] = v[r] > 0.f ? fmaxf(v[r], 0x1p-24f) : v[r];
    store_any<Z, V>(p, g.N - n, k);
  } else {
    store_any<Z, V>(p, g.N - n, v);
  }
}

// Bias, activation and residual of V neighbouring columns n .. n + V - 1 of row m; stores y and, if kept, z.
template <typename T, int V>
__device__ __forceinline__ void finish(const MatArgs& g, int m, int n, float (&v)[V], const AnyVec<T, V>& bias,
                                       const AnyVec<T, V>& res) {
  const int left = g.N - n;
  if (g.bias) {
#pragma unroll
    for (int r = 0; r < V; ++r) v[r] += (float)bias.e[r];
  }
  if (g.z) keep_z<typename ZOf<T>::type, V>(g, m, n, v);
  act_all<sizeof(T) == 4>(v, g.act, g.slope);
  if (g.res) {
#pragma unroll
    for (int r = 0; r < V; ++r) v[r] += (float)res.e[r];
  }
  store_any<T, V>(reinterpret_cast<T*>(g.c) + (size_t)m * g.ldc + n, left, v);
}

// ------------------------------------------------------------------------------------------------
// The tiled product.  A workgroup owns a BM x BN tile of C and walks the reduction in chunks of 128 bytes of a row
// (64 16-bit or 32 fp32 elements) through two LDS stages (four where memory has to be waited for, see launch_layout):
// chunk c + 1 travels while chunk c feeds the matrix cores, one barrier a chunk.  DMA: whole chunks go straight from
// memory to LDS (16-byte pieces, operands 16-byte aligned); the reduction's last, partial chunk, and every chunk of
// operands of another alignment, go through registers with masks.
//
// fp32 is bound by the matrix cores: 8192^3 at 139 TFLOP/s of the library's 154 (128-wide tiles); smaller ones lose
// to tiles that do not divide over the CUs and to the ends of short reductions, 2400 x 2560 -> 512 64 us = 98
// TFLOP/s.  16 bits with these tiles are bound by LDS and by the wait for a chunk: 2048^3 29 us = 590 TFLOP/s.
//
// LDS images of an operand with R rows in the tile:
//   k contiguous      [R][128 B], 16-byte pieces of a row XOR-ed with row & 7: the 16 rows a fragment load touches
//                     spread over all banks
//   index contiguous  [chunk][R elements]; 16-bit: 32-byte blocks XOR-ed with (k & 3) | (k >> 1 & 4), fp32: 64-byte
//                     blocks with 2 bits of k, so that the rows of k one fragment load touches fall on different banks
// 16-bit fragments of a column-major image come from ds_read_b64_tr_b16, which hands lane i of 16 the i-th column of a
// 4 x 16 block; fp32 fragments are single words.  The order of k inside a chunk only has to be the same for A and B.
// B is the MFMA's row operand, so a lane ends with four neighbouring columns of one row of C.
// ------------------------------------------------------------------------------------------------
template <int MODE, int R>
__device__ __forceinline__ int col_swizzle(int k) {       // in 16-byte pieces
  if (MODE == MODE_16) return (R >= 128 ? (k & 3) | ((k >> 1) & 4) : k & 3) << 1;   // (64: a row of k has four blocks)
  return ((MODE == MODE_F32 ? k >> 2 : k >> 3) & 3) << 2;
}

template <int MODE, bool KC, int R, int NT>
struct Operand {
  typedef typename ElemOf<MODE>::T T;
  static constexpr int ESZ = sizeof(T), EPP = 16 / ESZ, BK = 128 / ESZ;
  static constexpr int PIECES = (R * 8 + NT - 1) / NT;    // 16-byte pieces a thread stages (the last one: some waves)
  __device__ __forceinline__ static bool mine(int it, int thread) { return R * 8 % NT == 0 || it * NT + thread < R * 8; }
  static constexpr int PPR = R * ESZ / 16;                // pieces of a row of k (index contiguous)
  const char* src[PIECES];                                // this thread's pieces of chunk 0 (DMA)
  const char* base;
  long long ldb;                                          // bytes
  int o0, outer, K, tid;

  __device__ __forceinline__ void piece(int it, int& row, int& pc) const {   // tile row (of C or of k), source piece
    const int q = it * NT + tid;
    if (KC) {
      row = q >> 3;
      pc = (q & 7) ^ (row & 7);
    } else {
      row = q / PPR;
      pc = (q % PPR) ^ col_swizzle<MODE, R>(row);
    }
  }

  __device__ __forceinline__ void init(const void* p, long long ld, int o0_, int outer_, int K_, int tid_) {
    base = reinterpret_cast<const char*>(p);
    ldb = ld * ESZ;
    o0 = o0_;
    outer = outer_;
    K = K_;
    tid = tid_;
  }

  // addresses of chunk 0's pieces, clamped into the operand (rows and columns of C beyond its edge are computed from
  // repeated values and never stored)
  __device__ __forceinline__ void start() {
#pragma unroll
    for (int it = 0; it < PIECES; ++it) {
      int row, pc;
      piece(it, row, pc);
      if (KC) src[it] = base + (long long)min(o0 + row, outer - 1) * ldb + pc * 16;
      else src[it] = base + (long long)row * ldb + (long long)min(o0 + pc * EPP, outer - EPP) * ESZ;
    }
  }

  __device__ __forceinline__ void dma(char* stage, int c) {      // (a chunk's distance is uniform: no state but src)
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const long long at = c * (KC ? 128ll : BK * ldb);
#pragma unroll
    for (int it = 0; it < PIECES; ++it) {
      if (!mine(it, wave * 64)) continue;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src[it] + at),
                                       (__attribute__((address_space(3))) void*)(stage + (it * NT + wave * 64) * 16), 16,
                                       0, 0);
    }
  }

  __device__ __forceinline__ void fetch(int c, uint4 (&r)[PIECES]) const {
#pragma unroll
    for (int it = 0; it < PIECES; ++it) {
      int row, pc;
      piece(it, row, pc);
      r[it] = make_uint4(0, 0, 0, 0);
      const int o = o0 + (KC ? row : pc * EPP), k = c * BK + (KC ? pc * EPP : row);
      if (o >= outer || k >= K || !mine(it, tid)) continue;
      const int left = KC ? K - k : outer - o;            // elements of the piece that exist
      const char* p = base + (KC ? (long long)o * ldb + (long long)k * ESZ : (long long)k * ldb + (long long)o * ESZ);
      if (left >= EPP) {
        r[it] = reinterpret_cast<const Any16*>(p)->u;
      } else {
        Vec16<T> v;
#pragma unroll
        for (int e = 0; e < EPP; ++e) v.e[e] = e < left ? reinterpret_cast<const T*>(p)[e] : (T)0.f;
        r[it] = v.u;
      }
    }
  }

  __device__ __forceinline__ void put(char* stage, const uint4 (&r)[PIECES]) const {
#pragma unroll
    for (int it = 0; it < PIECES; ++it)
      if (mine(it, tid)) *reinterpret_cast<uint4*>(stage + (it * NT + tid) * 16) = r[it];
  }
};

// (The restrict gives the read alias information; without any the compiler waits for every LDS-DMA in flight before
// it.)
__device__ __forceinline__ s16x4 read_transposed(const char* __restrict__ p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}

// Fragment loads.  sub: first of the 16 rows or columns of C; lane = 16 g + lc.
template <bool KC, int R>
__device__ __forceinline__ bf16x8 frag16(const char* s, int sub, int kk, int lc, int g) {
  if (KC) return *reinterpret_cast<const bf16x8*>(s + (sub + lc) * 128 + (((kk * 4 + g) ^ (lc & 7)) << 4));
  const int k = kk * 32 + 8 * g + (lc >> 2);
  const char* p = s + k * (R * 2) + (((sub >> 3) ^ col_swizzle<MODE_16, R>(k)) << 4) + (lc & 3) * 8;
  union { s16x4 h[2]; bf16x8 v; } f;
  f.h[0] = read_transposed(p);
  f.h[1] = read_transposed(p + 4 * R * 2);
  return f.v;
}

template <bool KC, int R>
__device__ __forceinline__ f32x4 frag32(const char* s, int sub, int kk, int lc, int g) {   // k = 16 kk + 4 g + 0 .. 3
  if (KC) return *reinterpret_cast<const f32x4*>(s + (sub + lc) * 128 + (((kk * 4 + g) ^ (lc & 7)) << 4));
  f32x4 f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int k = kk * 16 + 4 * g + e;
    f[e] = *reinterpret_cast<const float*>(s + k * (R * 4) + (((sub >> 2) ^ col_swizzle<MODE_F32, R>(k)) << 4) + lc * 4);
  }
  return f;
}

template <bool KC, int R>
__device__ __forceinline__ void frag_split(const char* s, int sub, int lc, int g, bf16x8& hi, bf16x8& lo) {  // k = 8 g ...
  float v[8];
  if (KC) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 t = *reinterpret_cast<const f32x4*>(s + (sub + lc) * 128 + (((2 * g + h) ^ (lc & 7)) << 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * h + e] = t[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = 8 * g + e;
      v[e] = *reinterpret_cast<const float*>(s + k * (R * 4) + (((sub >> 2) ^ col_swizzle<MODE_S3, R>(k)) << 4) + lc * 4);
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const vca_e16 h = (vca_e16)v[e];
    hi[e] = h;
    lo[e] = (vca_e16)(v[e] - (float)h);
  }
}

// Workgroup -> tile.  Consecutive workgroups go to the 8 XCDs in turn; each XCD gets a contiguous range of the tiles,
// and those run through groups of 8 tile rows column by column, so the tiles an XCD's L2 holds share operands.
__device__ __forceinline__ void tile_of(const MatArgs& g, int id, int total, int& tm, int& tn, int& kz) {
  const int x = id & 7, per = total >> 3, rem = total & 7;
  int t = x * per + min(x, rem) + (id >> 3);
  const int tiles = g.ntm * g.ntn;
  kz = t / tiles;
  t -= kz * tiles;
  const int band = 8 * g.ntn, grp = t / band, m0 = grp * 8, rows = min(8, g.ntm - m0);
  t -= grp * band;
  tm = m0 + t % rows;
  tn = t / rows;
}

// The end of a tile.  A split reduction stores its partial tile as it is.  Otherwise the accumulators pass through
// LDS (fp32, 16-byte pieces of a row XOR-ed with the row) so that a thread finishes 16 bytes of a row of C and a wave
// writes whole lines, in as many parts as the tile is larger than the LDS of the two stages.
template <typename T, int BM, int BN, int NWM, int NWN>
__device__ __forceinline__ void store_tile(const MatArgs& g, const f32x4 (&acc)[BM / NWM / 16][BN / NWN / 16], char* smem,
                                           int m0, int n0, int kz, int wm, int wn, int lc, int lg, int tid) {
  constexpr int NT = NWM * NWN * 64, TM = BM / NWM / 16, TN = BN / NWN / 16;
  if (g.ksplit > 1) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int m = m0 + (wm * TM + i) * 16 + lc;
      if (m >= g.M) continue;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int n = n0 + (wn * TN + j) * 16 + 4 * lg;
        if (n < g.npad)
          *reinterpret_cast<f32x4*>(g.part + ((size_t)kz * g.M + m) * g.npad + n) = acc[i][j];
      }
    }
    return;
  }
  constexpr int V = 16 / (int)sizeof(T), TPR = BN / V;
  constexpr int PARTS = BM * BN * 4 > 2 * (BM + BN) * 128 ? BM * BN * 4 / (2 * (BM + BN) * 128) : 1, HM = TM / PARTS;
  constexpr int STEP = NT / TPR, ROWS = NWM * HM * 16, ITER = ROWS / STEP;   // a thread keeps its columns and takes
  static_assert(NT % TPR == 0 && ROWS % STEP == 0, "");                      // every STEP-th row
  const int col = (tid % TPR) * V, n = n0 + col;
  const AnyVec<T, V> bias = bias_of<T, V>(g, min(n, g.N));
#pragma unroll
  for (int h = 0; h < PARTS; ++h) {
    auto row_of = [&](int row) { return m0 + (row / (HM * 16) * TM + h * HM) * 16 + row % (HM * 16); };
    // All of the part's residual is asked for at once, under the turn through LDS.  The counter that loads and stores
    // share is in order, so a load between the rows' stores would wait for memory twice a row.
    AnyVec<T, V> res[ITER];
    if (g.res && n < g.N) {
#pragma unroll
      for (int k = 0; k < ITER; ++k) res[k] = res_of<T, V>(g, min(row_of(tid / TPR + k * STEP), g.M - 1), n);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < HM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int row = (wm * HM + i) * 16 + lc, pc = (wn * TN + j) * 4 + lg;
        *reinterpret_cast<f32x4*>(smem + row * (BN * 4) + ((pc ^ lc) << 4)) = acc[h * HM + i][j];
      }
    __syncthreads();
    if (n >= g.N) continue;
#pragma unroll 1
    for (int row = tid / TPR; row < ROWS; row += STEP) {
      const int m = row_of(row);
      if (m < g.M) {
        float v[V];
#pragma unroll
        for (int e = 0; e < V; e += 4) {
          const f32x4 t =
              *reinterpret_cast<const f32x4*>(smem + row * (BN * 4) + ((((col + e) >> 2) ^ (row & 15)) << 4));
#pragma unroll
          for (int r = 0; r < 4; ++r) v[e + r] = t[r];
        }
        finish<T, V>(g, m, n, v, bias, res[0]);
      }
#pragma unroll
      for (int k = 0; k + 1 < ITER; ++k) res[k] = res[k + 1];      // (a rolled loop: the rows share one copy of the code)
    }
  }
}

template <int MODE, bool AKC, bool BKC, int BM, int BN, int NWM, int NWN, bool DMA, int STAGES,
          bool TURN>
__device__ __forceinline__ void product_block(const MatArgs& g, int id, int total) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typedef typename ElemOf<MODE>::T T;
  constexpr int NT = NWM * NWN * 64, BK = 128 / (int)sizeof(T);
  constexpr int TM = BM / NWM / 16, TN = BN / NWN / 16;
  constexpr int STAGE = (BM + BN) * 128;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lc = lane & 15, lg = lane >> 4;
  const int wm = wave / NWN, wn = wave % NWN;
  int tm, tn, kz;
  tile_of(g, id, total, tm, tn, kz);
  const int m0 = tm * BM, n0 = tn * BN;
  const int c0 = kz * g.cpz, c1 = min((g.K + BK - 1) / BK, c0 + g.cpz);
  const int whole = DMA ? max(c0, min(c1, g.K / BK)) : c0;   // chunks [c0, whole) travel by DMA, the rest through registers

  Operand<MODE, AKC, BM, NT> A;
  Operand<MODE, BKC, BN, NT> B;
  A.init(g.a, g.lda, m0, g.M, g.K, tid);
  B.init(g.b, g.ldb, n0, g.N, g.K, tid);

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](const char* sa) {
    const char* sb = sa + BM * 128;
    if (MODE == MODE_16) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        bf16x8 fb[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[j] = frag16<BKC, BN>(sb, (wn * TN + j) * 16, kk, lc, lg);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const bf16x8 fa = frag16<AKC, BM>(sa, (wm * TM + i) * 16, kk, lc, lg);
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = VCA_MFMA_16x16x32(fb[j], fa, acc[i][j]);
        }
      }
    } else if (MODE == MODE_F32) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        f32x4 fb[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[j] = frag32<BKC, BN>(sb, (wn * TN + j) * 16, kk, lc, lg);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const f32x4 fa = frag32<AKC, BM>(sa, (wm * TM + i) * 16, kk, lc, lg);
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < TN; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[j][e], fa[e], acc[i][j], 0, 0, 0);
        }
      }
    } else {
      bf16x8 bh[TN], bl[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) frag_split<BKC, BN>(sb, (wn * TN + j) * 16, lc, lg, bh[j], bl[j]);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        bf16x8 ah, al;
        frag_split<AKC, BM>(sa, (wm * TM + i) * 16, lc, lg, ah, al);
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          if (MODE == MODE_S3) {
            acc[i][j] = VCA_MFMA_16x16x32(bl[j], ah, acc[i][j]);
            acc[i][j] = VCA_MFMA_16x16x32(bh[j], al, acc[i][j]);
          }
          acc[i][j] = VCA_MFMA_16x16x32(bh[j], ah, acc[i][j]);
        }
      }
    }
  };

  if (c0 < whole) {
    // TURN: each tile starts at a chunk of its own.  Where every CU walks through its rows of W at the same column
    // and the rows lie a power of two apart, few of the memory's channels are asked at a time (4096 -> 16384 in bf16,
    // 8 rows 29.8 -> 25.8 us, 64 rows 31.6 -> 27.5; with less than half the CUs at work it changes nothing).
    const int turn = TURN ? tn % (whole - c0) : 0;
    A.start();
    B.start();
    static_assert((STAGES & (STAGES - 1)) == 0, "");
    auto stage = [&](int c) { return smem + ((c - c0) & (STAGES - 1)) * STAGE; };
    auto send = [&](int c) {
      const int k = !TURN ? c : c + turn < whole ? c + turn : c + turn - (whole - c0);
      A.dma(stage(c), k);
      B.dma(stage(c) + BM * 128, k);
    };
    for (int c = c0; c < min(whole, c0 + STAGES - 1); ++c) send(c);
    for (int c = c0; c < whole; ++c) {
      // Chunk c has landed, in every wave behind the barrier: at most the STAGES - 2 chunks behind it are under way.
      // Every wave has left the stage that is sent to next, chunk c - 1's, with its reads done.
      if (STAGES > 2 && c + STAGES - 2 < whole) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * (A.PIECES + B.PIECES)) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
      }
      if (c + STAGES - 1 < whole) send(c + STAGES - 1);
      compute(stage(c));
    }
  }
  if (whole < c1) {                                       // not by DMA: chunk c + 1 waits in registers under chunk c
    uint4 ra[A.PIECES], rb[B.PIECES];
    A.fetch(whole, ra);
    B.fetch(whole, rb);
    __syncthreads();
    for (int c = whole; c < c1; ++c) {
      char* st = smem + ((c - whole) & 1) * STAGE;
      A.put(st, ra);
      B.put(st + BM * 128, rb);
      __syncthreads();                                    // (two stages: the writers of c + 1 need not wait for c)
      if (c + 1 < c1) {
        A.fetch(c + 1, ra);
        B.fetch(c + 1, rb);
      }
      compute(st);
    }
  }

  store_tile<T, BM, BN, NWM, NWN>(g, acc, smem, m0, n0, kz, wm, wn, lc, lg, tid);
}

template <int MODE, bool AKC, bool BKC, int BM, int BN, int NWM, int NWN, bool DMA, int STAGES, bool TURN>
__global__ __launch_bounds__(NWM * NWN * 64) void matmul_kernel(const MatArgs g) {
  product_block<MODE, AKC, BKC, BM, BN, NWM, NWN, DMA, STAGES, TURN>(g, blockIdx.x, gridDim.x);
}

// dx = dz W and dW = dz^T x in one launch, by 64 x 64 tiles: workgroups [0, first) take dx.
template <int MODE, bool DMA>
__global__ __launch_bounds__(256) void matmul_pair_kernel(const MatArgs x, const MatArgs w, int first) {
  if ((int)blockIdx.x < first) product_block<MODE, true, false, 64, 64, 2, 2, DMA, 2, false>(x, blockIdx.x, first);
  else product_block<MODE, false, false, 64, 64, 2, 2, DMA, 2, false>(w, blockIdx.x - first, gridDim.x - first);
}

// ------------------------------------------------------------------------------------------------
// The tiled product for large 16-bit ones: 256 x 256 tiles, eight waves of 128 x 64 each, two to a SIMD, one
// workgroup to a CU.  LDS carries 2 x 64 KB stages and feeds the waves 192 KB of fragments a chunk, under the time
// the matrix cores need for it.  The waves overlap by themselves: while the 32 MFMAs of one half chunk run, the 12
// fragments of the next half are read (the second half of chunk c, then the first of chunk c + 1) and, in the second
// half, a piece of chunk c + 2 is sent behind each row of MFMAs.  The chunk's only barrier sits in its middle: there
// every wave has its last fragments of chunk c in registers, chunk c + 1 has landed (it was sent a whole chunk
// earlier), and chunk c's stage is free to be refilled.
//
// Bound by the matrix cores: 8192^3 in bf16 at 1390 (x W^T), 1447 (dx) and 1465 TFLOP/s (dW), where the library's
// product reaches 1485; with few chunks a tile the pipeline's ends show, 8192 x 4096 x 4096: 1270, 1300, 1408.  Tried
// and slower: four waves of 128 x 128 (fewer fragment reads, but accumulators that do not fit the registers next to
// the fragments: 459 us against 339), touching the next chunk's lines in L2, the barrier shifted by a quarter chunk,
// chunks visited in an order that differs between tiles.
// ------------------------------------------------------------------------------------------------
template <bool KC>
struct WideOperand {
  static constexpr int NT = 512, PIECES = 4;
  const char* at;                     // the tile's first element of the next chunk to fetch: uniform
  long long step;                     // bytes a chunk
  unsigned off[PIECES];               // this thread's pieces, relative to it

  __device__ __forceinline__ void init(const void* p, long long ld, int o0, int outer, int c0, int tid) {
    const long long ldb = ld * 2;
    at = reinterpret_cast<const char*>(p) + (KC ? o0 * ldb + c0 * 128ll : c0 * 64 * ldb + o0 * 2ll);
    step = KC ? 128 : 64 * ldb;
#pragma unroll
    for (int it = 0; it < PIECES; ++it) {
      const int q = it * NT + tid;
      if (KC) {
        const int row = q >> 3;
        off[it] = (unsigned)(min(row, outer - 1 - o0) * (int)ldb + ((q & 7) ^ (row & 7)) * 16);
      } else {
        const int k = q >> 5, pc = (q & 31) ^ col_swizzle<MODE_16, 256>(k);
        off[it] = (unsigned)(k * (int)ldb + min(pc * 8, outer - 8 - o0) * 2);
      }
    }
  }

  __device__ __forceinline__ void dma(char* stage, int wave, int it) const {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(at + off[it]),
                                     (__attribute__((address_space(3))) void*)(stage + (it * NT + wave * 64) * 16), 16,
                                     0, 0);
  }
};

template <bool AKC, bool BKC>
__global__ __launch_bounds__(512) void matmul_wide_kernel(const MatArgs g) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int BM = 256, STAGE = 2 * BM * 128, TM = 8, TN = 4;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lc = lane & 15, lg = lane >> 4, wm = wave >> 2, wn = wave & 3;
  int tm, tn, kz;
  tile_of(g, blockIdx.x, gridDim.x, tm, tn, kz);
  const int m0 = tm * BM, n0 = tn * BM;
  const int c0 = kz * g.cpz, c1 = min((g.K + 63) / 64, c0 + g.cpz), whole = max(c0, min(c1, g.K / 64));

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // Fragment addresses as frag16's, but from one lane offset an operand: a fragment's place (sub = 16 i) is a constant
  // added where k is contiguous, a constant XOR-ed where it is not (a row of k has 16 blocks, i sits in the swizzled
  // bits), and so is kk the other way round.
  auto lane_off = [&](bool kc, int sub) {
    if (kc) return (unsigned)((sub + lc) * 128 + ((lg ^ (lc & 7)) << 4));
    const int k = 8 * lg + (lc >> 2);
    return (unsigned)(k * 512 + (((sub >> 4) ^ ((k & 3) | ((k >> 1) & 4))) << 5) + (lc & 3) * 8);
  };
  const unsigned oa = lane_off(AKC, wm * TM * 16), ob = lane_off(BKC, wn * TN * 16);
  auto read_frag = [&](bool kc, unsigned o, const char* image, int kk, int i) {
    if (kc) return *reinterpret_cast<const bf16x8*>(image + (o ^ (kk << 6)) + i * 2048);
    const char* p = image + (o ^ (i << 5)) + kk * 16384;
    union { s16x4 h[2]; bf16x8 v; } f;
    f.h[0] = read_transposed(p);
    f.h[1] = read_transposed(p + 2048);
    return f.v;
  };
  auto read_a = [&](const char* st, int kk, int i) { return read_frag(AKC, oa, st, kk, i); };
  auto read_b = [&](const char* st, int kk, int j) { return read_frag(BKC, ob, st + BM * 128, kk, j); };

  if (c0 < whole) {
    WideOperand<AKC> A;
    WideOperand<BKC> B;
    A.init(g.a, g.lda, m0, g.M, c0, tid);
    B.init(g.b, g.ldb, n0, g.N, c0, tid);
    auto send = [&](char* st, int it) {                   // one of the eight pieces a thread sends of a chunk
      if (it < 4) A.dma(st, wave, it);
      else B.dma(st + BM * 128, wave, it - 4);
      if (it == 7) {
        A.at += A.step;
        B.at += B.step;
      }
    };
    bf16x8 fa[TM], fb0[TN], fb1[TN];
#pragma unroll
    for (int it = 0; it < 8; ++it) send(smem, it);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (c0 + 1 < whole) {
#pragma unroll
      for (int it = 0; it < 8; ++it) send(smem + STAGE, it);
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) fb0[j] = read_b(smem, 0, j);
#pragma unroll
    for (int i = 0; i < TM; ++i) fa[i] = read_a(smem, 0, i);
    // One half chunk: its MFMAs row by row, and behind each row that row's fragment of the next half (half kk of stage
    // st) and, in the second half, one piece of the chunk after the next.
    auto half = [&](const bf16x8 (&fb)[TN], const char* st, int kk, bf16x8 (&nb)[TN], char* to, auto sends) {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if constexpr (decltype(sends)::value) send(to, i);
        if (i < TN) nb[i] = read_b(st, kk, i);
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = VCA_MFMA_16x16x32(fb[j], fa[i], acc[i][j]);
        fa[i] = read_a(st, kk, i);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // chunk c + 1 has landed, and chunk c's last fragments are in registers
    auto meet = [&]() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    int c = c0;
    for (; c + 2 < whole; ++c) {
      char* st = smem + ((c - c0) & 1) * STAGE;
      half(fb0, st, 1, fb1, nullptr, std::false_type());
      meet();
      half(fb1, smem + ((c - c0 + 1) & 1) * STAGE, 0, fb0, st, std::true_type());
    }
    for (; c < whole; ++c) {                              // the last two: nothing left to send
      half(fb0, smem + ((c - c0) & 1) * STAGE, 1, fb1, nullptr, std::false_type());
      meet();
      // (behind the last chunk this reads the other stage's old contents, which nothing uses)
      half(fb1, smem + ((c - c0 + 1) & 1) * STAGE, 0, fb0, nullptr, std::false_type());
    }
  }
  if (whole < c1) {                                       // the reduction's partial chunk, through registers
    Operand<MODE_16, AKC, BM, 512> A;
    Operand<MODE_16, BKC, BM, 512> B;
    A.init(g.a, g.lda, m0, g.M, g.K, tid);
    B.init(g.b, g.ldb, n0, g.N, g.K, tid);
    uint4 ra[A.PIECES], rb[B.PIECES];
    A.fetch(whole, ra);
    B.fetch(whole, rb);
    __syncthreads();
    A.put(smem, ra);
    B.put(smem + BM * 128, rb);
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      bf16x8 fb[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) fb[j] = read_b(smem, kk, j);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const bf16x8 fa = read_a(smem, kk, i);
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = VCA_MFMA_16x16x32(fb[j], fa, acc[i][j]);
      }
    }
  }
  store_tile<vca_e16, BM, BM, 2, 4>(g, acc, smem, m0, n0, kz, wm, wn, lc, lg, tid);
}

// C from the ksplit partial products, added in order of the reduction, through the same epilogue (workgroup `block` of
// `blocks`)
template <typename T>
__device__ __forceinline__ void fold_product(const MatArgs& g, int block, int blocks) {
  constexpr int V = 16 / (int)sizeof(T);
  const int nv = (g.N + V - 1) / V;
  const size_t total = (size_t)g.M * nv, slab = (size_t)g.M * g.npad;
  for (size_t i = (size_t)block * 256 + threadIdx.x; i < total; i += (size_t)blocks * 256) {
    const int m = (int)(i / nv), n = (int)(i - (size_t)m * nv) * V;
    const float* p = g.part + (size_t)m * g.npad + n;      // npad is a multiple of 8
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.f;
#pragma unroll 4
    for (int s = 0; s < g.ksplit; ++s)
#pragma unroll
      for (int e = 0; e < V; e += 4) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(p + s * slab + e);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[e + r] += t[r];
      }
    finish<T, V>(g, m, n, v, bias_of<T, V>(g, n), res_of<T, V>(g, m, n));
  }
}

// db[n] (+)= sum of the slabs: 16 columns a workgroup, each column's slabs in 16 interleaved runs
struct BiasArgs {
  const float* part;
  void* db;
  int N, slabs, add;
};

template <typename T>
__device__ __forceinline__ void fold_bias(const BiasArgs& b, int block, float (*red)[17]) {
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, n = block * 16 + tx;
  float t = 0.f;
  if (n < b.N) {
#pragma unroll 8
    for (int s = ty; s < b.slabs; s += 16) t += b.part[(size_t)s * b.N + n];
  }
  red[ty][tx] = t;
  __syncthreads();
  if (ty || n >= b.N) return;
#pragma unroll
  for (int y = 1; y < 16; ++y) t += red[y][tx];
  T* db = reinterpret_cast<T*>(b.db);
  db[n] = (T)(b.add ? t + (float)db[n] : t);
}

// What is left to add up behind a forward pass (one product) or a backward pass (two products and the bias gradient),
// in one launch: workgroups [0, first[1]) take product 0, [first[1], first[2]) product 1, the rest the bias gradient.
struct FoldArgs {
  MatArgs g[2];
  BiasArgs b;
  int first[4];
};

template <typename T>
__global__ __launch_bounds__(256) void fold_kernel(const FoldArgs f) {
  __shared__ float red[16][17];
  const int w = blockIdx.x;
  if (w < f.first[1]) fold_product<T>(f.g[0], w, f.first[1]);
  else if (w < f.first[2]) fold_product<T>(f.g[1], w - f.first[1], f.first[2] - f.first[1]);
  else fold_bias<T>(f.b, w - f.first[2], red);
}

// ------------------------------------------------------------------------------------------------
// Few rows (M <= 16, both operands with k contiguous): the product reads W once and does next to nothing with it, so
// there is no tile to share through LDS.  A workgroup owns 16 columns of C (and a range of the reduction where there
// are few columns); each lane streams 16 bytes of a W row, and of an x row out of the caches, straight into an MFMA
// operand. A wave takes two neighbouring chunks of 64 bytes at a time, so the line of each of its 16 rows is asked
// for by one wave in a row (31 us against 35 with single chunks dealt out to the waves, 4096 -> 16384 in bf16, 8
// rows), and the next two fly under this pair's products.  More in flight (four chunks: 32 us), 32 columns a
// workgroup (34) or four waves (33) were longer.  Bound by memory: 5.3 TB/s with one row, 4.9 with four (4096 ->
// 16384), whose x fragments pass through L2 as well: with more rows the tiles above take over (FEW_BYTES).  The
// waves' partial tiles meet in LDS.  Rows of x beyond M repeat the last one.
// ------------------------------------------------------------------------------------------------
constexpr int FEW_WAVES = 8, FEW_PAIR = 2, FEW_GROUP = FEW_WAVES * FEW_PAIR;

template <int MODE>
__global__ __launch_bounds__(FEW_WAVES * 64) void few_rows_kernel(const MatArgs g) {
  typedef typename ElemOf<MODE>::T T;
  constexpr int EPP = 16 / (int)sizeof(T), CK = 4 * EPP;   // elements a lane and a chunk take
  __shared__ f32x4 red[FEW_WAVES][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lc = lane & 15, lg = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const T* wp = reinterpret_cast<const T*>(g.b) + (long long)min(n0 + lc, g.N - 1) * g.ldb;
  const T* xp = reinterpret_cast<const T*>(g.a) + (long long)min(lc, g.M - 1) * g.lda;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  auto load = [&](const T* p, int c) {
    const int k = c * CK + lg * EPP;
    if (k + EPP <= g.K) return reinterpret_cast<const Any16*>(p + k)->u;
    Vec16<T> v;
#pragma unroll
    for (int e = 0; e < EPP; ++e) v.e[e] = k + e < g.K ? p[k + e] : (T)0.f;
    return v.u;
  };
  auto mul = [&](const uint4& uw, const uint4& ux) {
    if (MODE == MODE_16) {
      union { uint4 u; bf16x8 v; } w, x;
      w.u = uw;
      x.u = ux;
      acc = VCA_MFMA_16x16x32(w.v, x.v, acc);
    } else {
      union { uint4 u; float f[4]; } w, x;
      w.u = uw;
      x.u = ux;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(w.f[e], x.f[e], acc, 0, 0, 0);
    }
  };
  const int cb = blockIdx.y * g.cpz, ce = min((g.K + CK - 1) / CK, cb + g.cpz);   // this workgroup's chunks
  const int groups = (ce - cb - 1) / FEW_GROUP;            // groups of whole chunks (the last chunk is never in one)
  uint4 w[2][FEW_PAIR], x[2][FEW_PAIR];
  auto fetch = [&](int grp, int s) {
#pragma unroll
    for (int u = 0; u < FEW_PAIR; ++u) {
      const int k = (cb + grp * FEW_GROUP + wave * FEW_PAIR + u) * CK + lg * EPP;
      w[s][u] = reinterpret_cast<const Any16*>(wp + k)->u;
      x[s][u] = reinterpret_cast<const Any16*>(xp + k)->u;
    }
  };
  auto use = [&](int s) {
#pragma unroll
    for (int u = 0; u < FEW_PAIR; ++u) mul(w[s][u], x[s][u]);
  };
  if (groups > 0) fetch(0, 0);
  int q = 0;
  for (; q + 2 < groups; q += 2) {
    fetch(q + 1, 1);
    use(0);
    fetch(q + 2, 0);
    use(1);
  }
  if (q + 1 < groups) {
    fetch(q + 1, 1);
    use(0);
    use(1);
  } else if (q < groups) {
    use(0);
  }
  for (int c = cb + groups * FEW_GROUP + wave; c < ce; c += FEW_WAVES) mul(load(wp, c), load(xp, c));
  red[wave][lane] = acc;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int v = 1; v < FEW_WAVES; ++v) acc += red[v][lane];
  const int n = n0 + 4 * lg;
  if (lc >= g.M || n >= g.N) return;
  if (g.ksplit > 1) {
    *reinterpret_cast<f32x4*>(g.part + ((size_t)blockIdx.y * g.M + lc) * g.npad + n) = acc;
    return;
  }
  float v[4] = {acc[0], acc[1], acc[2], acc[3]};
  finish<T, 4>(g, lc, n, v, bias_of<T, 4>(g, n), res_of<T, 4>(g, lc, n));
}

// ------------------------------------------------------------------------------------------------
// dz = gy act'(z) and the columns' sums of it.  dz is rounded to the tensors' type because it is an operand of the two
// products behind it: the gradients of 16-bit layers carry its rounding beside their own (8192 x 4096 bf16: 0.0024 of
// their size instead of 0.0017), and two operands for its high and low part would double those products.
// A workgroup takes a strip of 32 x 16 bytes of columns and a range of rows (8 at a time); its column sums (of the unrounded dz, fp32) go to a slab, slabs are added in order.  Bound by
// memory: 8192 x 4096 bf16, gelu: 39 us, 5.1 TB/s.
// ------------------------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void act_bwd_kernel(int M, int N, int act, float slope, const T* __restrict__ gy,
                                                      const typename ZOf<T>::type* __restrict__ z, T* __restrict__ dz,
                                                      float* __restrict__ part, int rows, T* __restrict__ db,
                                                      int db_add) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ float red[8][32 * V];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int n = (blockIdx.x * 32 + tx) * V;
  const int r0 = blockIdx.y * rows, r1 = min(M, r0 + rows);
  float s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = 0.f;
  if (n + V <= N) {
    for (int r = r0 + ty; r < r1; r += 8) {
      const size_t o = (size_t)r * N + n;
      Vec16<T> a, d;
      AnyVec<typename ZOf<T>::type, V> b;
      a.u = reinterpret_cast<const Any16*>(gy + o)->u;
      if (z) b.load(z + o);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float v = (float)a.e[e];
        if (z) v *= act_slope<sizeof(T) == 4>((float)b.e[e], act, slope);
        s[e] += v;
        d.e[e] = (T)v;
      }
      if (dz) reinterpret_cast<Any16*>(dz + o)->u = d.u;
    }
  } else if (n < N) {
    for (int r = r0 + ty; r < r1; r += 8) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (n + e < N) {
          const size_t o = (size_t)r * N + n + e;
          float v = (float)gy[o];
          if (z) v *= act_slope<sizeof(T) == 4>((float)z[o], act, slope);
          s[e] += v;
          if (dz) dz[o] = (T)v;
        }
    }
  }
  if (!db) return;
#pragma unroll
  for (int e = 0; e < V; ++e) red[ty][tx * V + e] = s[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V; i += 256) {
    float t = 0.f;
#pragma unroll
    for (int y = 0; y < 8; ++y) t += red[y][i];
    const int col = blockIdx.x * 32 * V + i;
    if (col >= N) continue;
    if (gridDim.y > 1) part[(size_t)blockIdx.y * N + col] = t;
    else db[col] = (T)(db_add ? t + (float)db[col] : t);      // the only slab
  }
}

// ------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------
bool act_ok(int act) { return (act >= VCA_ACT_NONE && act <= VCA_ACT_SILU) && act != VCA_ACT_PRELU; }

int mode_of(const vca_matmul_desc& d) {
  if (d.type == VCA_T_F32) return d.nsplit == 0 ? MODE_F32 : d.nsplit == 3 ? MODE_S3 : d.nsplit == 1 ? MODE_S1 : -1;
  return d.type == (VCA_ELEM_TYPE ? VCA_T_F16 : VCA_T_BF16) && d.nsplit == 1 ? MODE_16 : -1;
}

struct Plan {
  MatArgs g;
  int mode, bm, bn;                   // the tile; 0: few rows
  bool dma, wide, low, tall;          // may be taken: the 256-wide tiles, the 32-row ones and four stages, those with more
                                      // rows than columns
  bool pair;                          // only the 64 x 64 tiles may
};

// Rows of x times bytes of W up to which few_rows_kernel takes a product of at most 16 rows: every workgroup of 16
// columns reads x again, a tile of 64 columns a quarter of that.  us, few_rows_kernel and tiles: bf16 4096 -> 16384,
// 1 row 25.1 / 26.2, 4 rows 27.6 / 26, 8 rows 31 / 25.8, 16 rows 39 / 26; 4096 -> 4096, 8 rows 10.2 / 11.9; fp32 4096
// -> 4096, 16 rows 25 / 21; 512 -> 512, 16 rows 4.2 / 6.6.
constexpr double FEW_BYTES = 500e6;
constexpr int LOW_ROWS = 128;         // see launch_layout

// Tile and split of a product, by the time the candidates would take.  A tile's chunk costs a CU `work` us of its
// matrix cores; a workgroup that has a CU to itself cannot go below `wait` us a chunk (LDS and memory latency, one
// barrier a chunk), a CU with r workgroups takes max(wait, r work), and all of them together no less than the
// operands' trip from memory.  `ends`: filling the pipeline and storing the tile.  A split adds one launch and a pass
// over the partial products.
// The four numbers of each tile were fitted to launches of 2 to 2000 us on this part; the choice is within some 10 % of
// the best one measured at each.  Where sides change (us):
//   fp32 8192 x 4096 <- 4096       64 wide 2349, 128 wide 2043
//   fp32 tall tiles                4800 x 1280 <- 512    128 x 64  63, 64 x 64  69
//                                  4800 x 512 <- 1280     80 x 64  62, 64 x 64  73
//                                  900 x 1300 <- 700      tall     23, 64 x 64  29
//                                  2400 x 512 <- 2560    160 x 64 split four ways 65, 128 x 128 split three ways 68
//                                  but 1500 x 2048 <- 2048  80 x 64 147, 64 x 64 114
//   16 bits 2048^3                 64 wide 29, 128 wide 30, 256 wide 39 (split)
//   16 bits 4800 x 2560 <- 5120    64 wide 197, 128 wide 137, 256 wide 112
//   16 bits 64 x 4096 <- 4096      64 wide 23, the same split four ways 13
//   16 bits 4800 x 1280 <- 512     tall tiles 11.9, 64 wide 13.6: too little for forms of their own
//   32 x 4096 <- 4096              32 x 64 tiles 12.2, 64 x 64 13.5; fp32 21.3 and 25.8
struct TileCost { int bm, bn; double work, wait, ends; };
constexpr TileCost COST[4][6] = {
    {{256, 256, 1.55, 1.55, 8.}, {128, 128, 0.53, 0.85, 2.}, {64, 64, 0.20, 0.45, 0.8}, {32, 64, 0.12, 0.24, 2.}},   // 16 bits
    {{128, 128, 1.95, 2.15, 5.5}, {64, 64, 0.56, 0.62, 2.}, {32, 64, 0.22, 0.44, 2.},                          // fp32, exact
     {160, 64, 1.22, 1.50, 4.5}, {128, 64, 1.05, 1.15, 3.3}, {80, 64, 0.73, 0.82, 2.}},
    {{128, 128, 0.92, 1.15, 4.}, {64, 64, 0.36, 0.55, 1.}, {32, 64, 0.15, 0.40, 2.},                  // fp32, three products
     {160, 64, 0.68, 1.05, 4.}, {128, 64, 0.63, 0.87, 2.3}},
    {{128, 128, 0.46, 0.85, 2.5}, {64, 64, 0.22, 0.45, 1.}, {32, 64, 0.12, 0.35, 2.}}};                 // fp32, one product

bool pick(Plan& p, int nc) {
  MatArgs& g = p.g;
  const double memory = ((double)g.M + g.N) * g.K * (p.mode == MODE_16 ? 2 : 4) / 5e6;   // both operands once, at 5 TB/s
  double best = 0.;
  p.bm = 0;
  for (const TileCost& t : COST[p.mode]) {
    if (!t.bm || (p.pair && t.bm != 64) || (t.bm == 256 && !p.wide) || (t.bm == 32 && !(p.low && g.M <= 32)) ||
        (t.bm > t.bn && !p.tall))
      continue;
    const long long tiles = ((g.M + (long long)t.bm - 1) / t.bm) * ((g.N + (long long)t.bn - 1) / t.bn);
    if (tiles >= (1 << 24)) continue;
    const double wait = t.wait * (p.low && g.M <= 64 && t.bm == 64 && p.mode == MODE_16 ? 0.75 : 1.);   // (four stages)
    for (int ks = 1; ks <= 32 && ks <= nc; ++ks) {
      const int chunks = (nc + ks - 1) / ks;
      if (ks > 1 && (chunks < 2 || tiles * ks > 2048)) break;
      const double r = (double)((tiles * ks + 255) / 256);
      double us = chunks * (r * t.work > wait ? r * t.work : wait);
      if (us < memory) us = memory;
      us += r * t.ends;
      if (ks > 1) us += 3. + (double)ks * g.M * g.npad * 1e-6;                 // written and read at 8 bytes / ps
      if (p.bm && us >= best) continue;
      best = us;
      p.bm = t.bm;
      p.bn = t.bn;
      g.cpz = chunks;
    }
  }
  if (!p.bm) return false;
  g.ksplit = (nc + g.cpz - 1) / g.cpz;
  g.ntm = (g.M + p.bm - 1) / p.bm;
  g.ntn = (g.N + p.bn - 1) / p.bn;
  return true;
}

int plan_of(const vca_matmul_desc* dp, const void* a, const void* b, Plan& p, bool pair = false) {
  VCA_CHECK_ARG(dp);
  const vca_matmul_desc& d = *dp;
  p.mode = mode_of(d);
  p.pair = pair;
  VCA_CHECK_ARG(p.mode >= 0 && d.M > 0 && d.N > 0 && d.K > 0 && act_ok(d.act));
  VCA_CHECK_ARG(d.M <= (1 << 30) && d.N <= (1 << 30) && d.K <= (1 << 30));   // (tile edges stay in an int)
  VCA_CHECK_ARG(!(d.a_col && !d.b_col));                   // no product here reads only its rows by columns
  const int esz = d.type == VCA_T_F32 ? 4 : 2, bk = 128 / esz;
  VCA_CHECK_ARG(d.lda >= (d.a_col ? d.M : (d.M > 1 ? d.K : 0)) && d.ldb >= (d.b_col ? d.N : (d.N > 1 ? d.K : 0)) &&
                d.ldc >= (d.M > 1 ? d.N : 0) && d.ldr >= 0);
  MatArgs& g = p.g;
  g.M = d.M;
  g.N = d.N;
  g.K = d.K;
  g.lda = d.lda;
  g.ldb = d.ldb;
  g.ldc = d.ldc;
  g.ldr = d.ldr;
  g.act = d.act;
  g.slope = d.slope;
  g.npad = (d.N + 7) / 8 * 8;
  g.part = nullptr;
  g.ksplit = 1;
  g.cpz = (d.K + bk - 1) / bk;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) |
                         (uintptr_t)(d.lda * esz) | (uintptr_t)(d.ldb * esz);
  const int per16 = 16 / esz;
  p.dma = (bits & 15) == 0 && (!d.a_col || d.M % per16 == 0) && (!d.b_col || d.N % per16 == 0);
  const double wbytes = (double)d.N * d.K * esz;
  if (d.M <= 16 && d.N <= (1 << 26) && !d.a_col && !d.b_col && (p.mode == MODE_16 || p.mode == MODE_F32) &&
      d.M * wbytes <= FEW_BYTES) {
    // A workgroup streams its 16 rows of W at some 30 GB/s, all of them at most at 5 TB/s; where columns alone give
    // too few of them to load the memory, the reduction is split too, if that saves more than the launch that adds
    // the parts (one row, split and unsplit: bf16 16384 -> 1024 12.9 / 21.7 us, fp32 2560 -> 512 7.2 / 9.6, fp32
    // 4096^2 21.2 / 20.3).
    p.bm = 0;
    const int nc = (d.K * esz + 63) / 64, blocks = (d.N + 15) / 16;
    double best = 0.;
    for (int ks = 1; ks <= 16 && (ks == 1 || (blocks * ks <= 512 && nc / ks >= 2 * FEW_GROUP)); ++ks) {
      const int chunks = (nc + ks - 1) / ks;
      const double stream = chunks * 1024. / 30e3, memory = wbytes / 5e6;
      const double us = (stream > memory ? stream : memory) + (ks > 1 ? 4. : 0.);
      if (ks == 1 || us < best) {
        best = us;
        g.cpz = chunks;
      }
    }
    g.ksplit = (nc + g.cpz - 1) / g.cpz;
    return 0;
  }
  // the 256-wide kernel addresses its pieces by 32-bit offsets from the tile: 256 rows (64 of k) of at most 4 MB
  p.low = p.dma && d.M <= LOW_ROWS && !d.a_col && !d.b_col;
  p.tall = p.dma && !d.a_col;
  p.wide = p.mode == MODE_16 && p.dma && d.lda <= (1 << 21) && d.ldb <= (1 << 21);
  return pick(p, g.cpz) ? 0 : -22;
}

template <int MODE, bool AKC, bool BKC, int BM, int BN, int NWM, bool DMA, int STAGES, bool TURN = false>
int launch_kernel(const Plan& p, hipStream_t s) {
  constexpr int LDS = STAGES * (BM + BN) * 128;            // at most 64 KB
  static_assert(LDS <= 64 * 1024, "");
  hipLaunchKernelGGL((matmul_kernel<MODE, AKC, BKC, BM, BN, NWM, 4 / NWM, DMA, STAGES, TURN>),
                     dim3(p.g.ntm * p.g.ntn * p.g.ksplit), dim3(256), LDS, s, p.g);
  return vca_launch_status();
}

template <int MODE, bool AKC, bool BKC>
int launch_layout(const Plan& p, hipStream_t s) {
  if (MODE == MODE_16 && p.bm == 256) {
    VCA_MAX_LDS((matmul_wide_kernel<AKC, BKC>));
    hipLaunchKernelGGL((matmul_wide_kernel<AKC, BKC>), dim3(p.g.ntm * p.g.ntn * p.g.ksplit), dim3(512), 128 * 1024, s, p.g);
    return vca_launch_status();
  }
  const bool turn = p.g.ksplit == 1 && p.g.ntm * p.g.ntn >= 128;
  if constexpr (AKC && BKC) {
    if (p.bm == 32)
      return turn ? launch_kernel<MODE, true, true, 32, 64, 1, true, 4, true>(p, s)
                  : launch_kernel<MODE, true, true, 32, 64, 1, true, 4>(p, s);
  }
  if constexpr (AKC && (MODE == MODE_F32 || MODE == MODE_S3)) {
    if (p.bm == 160) return launch_kernel<MODE, true, BKC, 160, 64, 2, true, 2>(p, s);
    if (p.bm == 128 && p.bn == 64) return launch_kernel<MODE, true, BKC, 128, 64, 2, true, 2>(p, s);
  }
  if constexpr (AKC && MODE == MODE_F32) {
    if (p.bm == 80) return launch_kernel<MODE, true, BKC, 80, 64, 1, true, 2>(p, s);
  }
  if (p.bm == 128)
    return p.dma ? launch_kernel<MODE, AKC, BKC, 128, 128, 2, true, 2>(p, s)
                 : launch_kernel<MODE, AKC, BKC, 128, 128, 2, false, 2>(p, s);
  if (!p.dma) return launch_kernel<MODE, AKC, BKC, 64, 64, 2, false, 2>(p, s);
  // Up to 128 rows the weights come from memory, not from another workgroup's lines in L2: three chunks under way
  // instead of one (16 bits 4096 -> 16384, 64 rows: 38 us against 40, 128: 48 against 56; fp32 4096^2, 64: 28 against
  // 32).  Larger products only lose workgroups a CU by it (2000 x 2048 -> 512: 15.5 against 14.9), column-major
  // operands too (64 x 4096 x 4096, dx: 15.5 against 13.6).
  if constexpr (AKC && BKC) {
    if (p.low)
      return turn ? launch_kernel<MODE, true, true, 64, 64, 2, true, 4, true>(p, s)
                  : launch_kernel<MODE, true, true, 64, 64, 2, true, 4>(p, s);
  }
  return launch_kernel<MODE, AKC, BKC, 64, 64, 2, true, 2>(p, s);
}

template <int MODE>
int launch_mode(const Plan& p, bool a_col, bool b_col, hipStream_t s) {
  if (a_col) return launch_layout<MODE, false, false>(p, s);
  if (b_col) return launch_layout<MODE, true, false>(p, s);
  return launch_layout<MODE, true, true>(p, s);
}

long long ws_of(const Plan& p) {
  return p.g.ksplit > 1 ? (long long)p.g.ksplit * p.g.M * p.g.npad : 0;
}

// Workspace floats of a product whatever its operands' alignment and strides, so that a caller may ask once a size.
long long ws_floats_of(const vca_matmul_desc* d, bool pair) {
  Plan p;
  if (plan_of(d, nullptr, nullptr, p) != 0) return 0;
  if (!p.bm) return ws_of(p);
  long long n = 0;
  const int nc = (p.g.K * (d->type == VCA_T_F32 ? 4ll : 2ll) + 127) / 128;
  const bool low = d->M <= LOW_ROWS && !d->a_col && !d->b_col;
  for (int form = 0; form < 3 + pair; ++form) {                   // not by DMA, by DMA, with the 256-wide tiles, in a pair
    p.low = (form == 1 || form == 2) && low;
    p.tall = (form == 1 || form == 2) && !d->a_col;
    p.wide = form == 2 && p.mode == MODE_16;
    p.pair = form == 3;
    if (pick(p, nc) && ws_of(p) > n) n = ws_of(p);
  }
  return n;
}

int z_type(int type) { return type == VCA_T_BF16 ? VCA_T_F16 : VCA_T_F32; }

bool aligned(int type, std::initializer_list<const void*> ps) {
  uintptr_t bits = 0;
  for (const void* p : ps) bits |= reinterpret_cast<uintptr_t>(p);
  return (bits & (type == VCA_T_F32 ? 3 : 1)) == 0;
}

void bind(MatArgs& g, const void* a, const void* b, const void* bias, const void* res, void* c, void* z, float* ws) {
  g.a = a;
  g.b = b;
  g.bias = bias;
  g.res = res;
  g.c = c;
  g.z = z;
  g.part = g.ksplit > 1 ? ws : nullptr;
}

// The product itself: into C, or into its partial products in ws where the plan splits it.
int launch_product(Plan& p, const vca_matmul_desc& d, const void* a, const void* b, const void* bias, const void* res,
                   void* c, void* z, float* ws, hipStream_t s) {
  MatArgs& g = p.g;
  bind(g, a, b, bias, res, c, z, ws);
  const bool ac = d.a_col != 0, bc = d.b_col != 0;
  if (p.bm == 0) {
    const dim3 grid((g.N + 15) / 16, g.ksplit);
    if (p.mode == MODE_16) hipLaunchKernelGGL(few_rows_kernel<MODE_16>, grid, dim3(FEW_WAVES * 64), 0, s, g);
    else hipLaunchKernelGGL(few_rows_kernel<MODE_F32>, grid, dim3(FEW_WAVES * 64), 0, s, g);
    return vca_launch_status();
  }
  switch (p.mode) {
    case MODE_16: return launch_mode<MODE_16>(p, ac, bc, s);
    case MODE_F32: return launch_mode<MODE_F32>(p, ac, bc, s);
    case MODE_S3: return launch_mode<MODE_S3>(p, ac, bc, s);
    default: return launch_mode<MODE_S1>(p, ac, bc, s);
  }
}

int grid_of(const Plan& p) { return p.g.ntm * p.g.ntn * p.g.ksplit; }

// Whether both products of a backward pass go by one launch, side by side instead of one after the other (us, one
// launch and two, with dz and db: bf16 300 x 512 x 512 11.6 / 16.2, 1801 x 1111 x 677 43 / 57; fp32 1000^3 52 / 63,
// 5000 x 1111 x 1333 377 / 373).
bool in_pair(const Plan& x, const Plan& w) {
  return x.bm == 64 && x.bn == 64 && w.bm == 64 && w.bn == 64 && x.dma == w.dma && grid_of(x) <= (1 << 22) &&
         grid_of(w) <= (1 << 22);
}

// Plans of both.  Other tiles are given up for one launch if the whole of it fits the CUs at once (600^3 fp32 27.3 ->
// 23.6; 4800 x 512 x 1280, 1080 workgroups, would go 137 -> 157).  Both products are always planned, wanted or not,
// so that dx does not depend on whether dW is formed too.
int plan_pair(const vca_linear_bwd& b, const vca_matmul_desc& x, const vca_matmul_desc& w, const void* dz, Plan& px, Plan& pw) {
  const int ex = plan_of(&x, dz, b.w, px), ew = plan_of(&w, dz, b.x, pw);
  if (ex && b.dx) return ex;
  if (ew && b.dw) return ew;
  if (ex || ew || in_pair(px, pw)) return 0;
  Plan qx, qw;
  if (plan_of(&x, dz, b.w, qx, true) || plan_of(&w, dz, b.x, qw, true)) return 0;
  if (in_pair(qx, qw) && grid_of(qx) + grid_of(qw) <= 512) {
    px = qx;
    pw = qw;
  }
  return 0;
}

template <int MODE>
int launch_pair_mode(const Plan& x, const Plan& w, hipStream_t s) {
  const int first = grid_of(x);
  const dim3 grid(first + grid_of(w));
  constexpr int LDS = 2 * 128 * 128;
  if (x.dma) hipLaunchKernelGGL((matmul_pair_kernel<MODE, true>), grid, dim3(256), LDS, s, x.g, w.g, first);
  else hipLaunchKernelGGL((matmul_pair_kernel<MODE, false>), grid, dim3(256), LDS, s, x.g, w.g, first);
  return vca_launch_status();
}

int launch_pair(const Plan& x, const Plan& w, hipStream_t s) {
  switch (x.mode) {
    case MODE_16: return launch_pair_mode<MODE_16>(x, w, s);
    case MODE_F32: return launch_pair_mode<MODE_F32>(x, w, s);
    case MODE_S3: return launch_pair_mode<MODE_S3>(x, w, s);
    default: return launch_pair_mode<MODE_S1>(x, w, s);
  }
}

void clear(FoldArgs& f) {
  f.first[0] = f.first[1] = f.first[2] = f.first[3] = 0;
  f.b = {nullptr, nullptr, 0, 0, 0};
}

// Adds up what is split: up to two products and the bias gradient in f.b (slabs 0: none).
int launch_folds(FoldArgs& f, const MatArgs* g0, const MatArgs* g1, int type, hipStream_t s) {
  auto blocks = [&](const MatArgs& g) {
    const long long n = ((long long)g.M * (g.npad / (type == VCA_T_F32 ? 4 : 8)) + 255) / 256;
    return (int)(n > 4096 ? 4096 : n);
  };
  if (g0) f.g[0] = *g0;
  if (g1) f.g[1] = *g1;
  f.first[1] = g0 ? blocks(*g0) : 0;
  f.first[2] = f.first[1] + (g1 ? blocks(*g1) : 0);
  f.first[3] = f.first[2] + (f.b.slabs ? (f.b.N + 15) / 16 : 0);
  if (!f.first[3]) return 0;
  if (type == VCA_T_F32) hipLaunchKernelGGL(fold_kernel<float>, dim3(f.first[3]), dim3(256), 0, s, f);
  else hipLaunchKernelGGL(fold_kernel<vca_e16>, dim3(f.first[3]), dim3(256), 0, s, f);
  return vca_launch_status();
}

int act_rows(int M, int N, int esz) {                     // rows a workgroup of act_bwd_kernel takes
  const long long strips = ((long long)N * esz + 511) / 512;
  int rows = M <= 16 ? 16 : 8;     // up to 16 rows one slab, and no launch to add slabs up (16 x 512: 3.9 us, 4.9 with two)
  auto slabs = [&]() { return ((long long)M + rows - 1) / rows; };
  while ((rows < 256 && strips * slabs() > 1024) || slabs() > 65535) rows *= 2;   // (65535: the grid's second dimension)
  return rows;
}

}  // namespace

extern "C" long long vca_matmul_act_ws_floats(const vca_matmul_desc* d) {
  return ws_floats_of(d, false);
}

extern "C" int vca_matmul_act(const vca_matmul_desc* d, const void* a, const void* b, const void* bias, const void* res,
                              void* c, void* z, float* ws, long long ws_floats, void* stream) {
  Plan p;
  VCA_CHECK_ARG(a && b && c);
  const int rc = plan_of(d, a, b, p);
  if (rc) return rc;
  VCA_CHECK_ARG(aligned(d->type, {a, b, bias, res, c}) && aligned(z_type(d->type), {z}));
  VCA_CHECK_ARG(ws_of(p) == 0 || (ws && ws_floats >= ws_of(p) && (reinterpret_cast<uintptr_t>(ws) & 15) == 0));
  const int e = launch_product(p, *d, a, b, bias, res, c, z, ws, (hipStream_t)stream);
  FoldArgs f;
  clear(f);
  return e ? e : launch_folds(f, p.g.ksplit > 1 ? &p.g : nullptr, nullptr, d->type, (hipStream_t)stream);
}

static long long act_bwd_ws(int type, int M, int N) {
  const int rows = act_rows(M, N, type == VCA_T_F32 ? 4 : 2);
  return ((long long)M + rows - 1) / rows * N;
}

// Launches dz and the slabs of db; leaves in f what of db is left to add up.
static int act_bwd(int type, int M, int N, int act, float slope, const void* gy, const void* z, void* dz, void* db,
                   int db_add, float* ws, FoldArgs& f, hipStream_t s) {
  const int esz = type == VCA_T_F32 ? 4 : 2, rows = act_rows(M, N, esz), slabs = (int)(((long long)M + rows - 1) / rows);
  const dim3 grid((unsigned)(((long long)N * esz + 511) / 512), (unsigned)slabs);
  if (esz == 4)
    hipLaunchKernelGGL(act_bwd_kernel<float>, grid, dim3(256), 0, s, M, N, act, slope, (const float*)gy, (const float*)z,
                       (float*)dz, ws, rows, (float*)db, db_add);
  else
    hipLaunchKernelGGL(act_bwd_kernel<vca_e16>, grid, dim3(256), 0, s, M, N, act, slope, (const vca_e16*)gy,
                       (const vca_z16*)z, (vca_e16*)dz, ws, rows, (vca_e16*)db, db_add);
  if (db && slabs > 1) f.b = {ws, db, N, slabs, db_add};
  return vca_launch_status();
}

static bool act_bwd_ok(int type, int M, int N, int act, const void* gy, const void* z, const void* dz, const void* db) {
  const int own16 = VCA_ELEM_TYPE ? VCA_T_F16 : VCA_T_BF16;
  return (type == VCA_T_F32 || type == own16) && M > 0 && N > 0 && act_ok(act) && gy && (act == VCA_ACT_NONE) == !z &&
         (!dz || z) && aligned(type, {gy, dz, db}) && aligned(z_type(type), {z});
}

// The three products' descriptors of a backward pass.
static vca_matmul_desc bwd_dx(const vca_linear_bwd& b) {
  vca_matmul_desc d = {b.M, b.K, b.N, b.type, b.nsplit, 0, 1, VCA_ACT_NONE, 0.f, b.N, b.ldw, b.K, 0};
  return d;
}

static vca_matmul_desc bwd_dw(const vca_linear_bwd& b) {
  vca_matmul_desc d = {b.N, b.K, b.M, b.type, b.nsplit, 1, 1, VCA_ACT_NONE, 0.f, b.N, b.ldx, b.K, b.K};
  return d;
}

static long long up4(long long n) { return (n + 3) / 4 * 4; }   // each part of the workspace starts at 16 bytes

extern "C" long long vca_linear_act_bwd_ws_floats(const vca_linear_bwd* b) {
  if (!b || b->M <= 0 || b->N <= 0 || b->K <= 0) return 0;
  const vca_matmul_desc x = bwd_dx(*b), w = bwd_dw(*b);
  return up4(act_bwd_ws(b->type, b->M, b->N)) + up4(ws_floats_of(&x, true)) + ws_floats_of(&w, true);
}

extern "C" int vca_linear_act_bwd(const vca_linear_bwd* b, float* ws, long long ws_floats, void* stream) {
  VCA_CHECK_ARG(b && b->K > 0 && act_bwd_ok(b->type, b->M, b->N, b->act, b->gy, b->z, b->dz, b->db));
  VCA_CHECK_ARG((!b->dx || b->w) && (!b->dw || b->x) && (b->act == VCA_ACT_NONE || b->dz || !(b->dx || b->dw)));
  VCA_CHECK_ARG(aligned(b->type, {b->x, b->w, b->dx, b->dw}));
  // (everything is checked before the first launch: a refused call has written nothing)
  const vca_matmul_desc x = bwd_dx(*b), w = bwd_dw(*b);
  const void* dz = b->dz ? b->dz : b->gy;
  Plan px, pw;
  px.g.ksplit = pw.g.ksplit = 1;
  if (b->dx || b->dw) {
    const int rc = plan_pair(*b, x, w, dz, px, pw);
    if (rc) return rc;
    if (!b->dx) px.g.ksplit = 1;                           // (nothing of it to add up)
    if (!b->dw) pw.g.ksplit = 1;
  }
  // one part of the workspace for each of db, dx and dw, so that what is split is added up by one launch at the end
  const long long at_x = b->db ? up4(act_bwd_ws(b->type, b->M, b->N)) : 0;
  const long long at_w = at_x + (b->dx ? up4(ws_of(px)) : 0), need = at_w + (b->dw ? ws_of(pw) : 0);
  VCA_CHECK_ARG(ws_floats >= need && (!need || (ws && (reinterpret_cast<uintptr_t>(ws) & 15) == 0)));
  hipStream_t s = (hipStream_t)stream;
  FoldArgs f;
  clear(f);
  int e = 0;
  if (b->dz || b->db) e = act_bwd(b->type, b->M, b->N, b->act, b->slope, b->gy, b->z, b->dz, b->db, b->db_add, ws, f, s);
  const void* old = b->dw_add ? b->dw : nullptr;
  if (!e && b->dx && b->dw && in_pair(px, pw)) {
    bind(px.g, dz, b->w, nullptr, nullptr, b->dx, nullptr, ws + at_x);
    bind(pw.g, dz, b->x, nullptr, old, b->dw, nullptr, ws + at_w);
    e = launch_pair(px, pw, s);
  } else {
    if (!e && b->dx) e = launch_product(px, x, dz, b->w, nullptr, nullptr, b->dx, nullptr, ws + at_x, s);
    if (!e && b->dw) e = launch_product(pw, w, dz, b->x, nullptr, old, b->dw, nullptr, ws + at_w, s);
  }
  return e ? e : launch_folds(f, px.g.ksplit > 1 ? &px.g : nullptr, pw.g.ksplit > 1 ? &pw.g : nullptr, b->type, s);
}
