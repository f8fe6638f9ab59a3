// Global norm of many gradient tensors, clipping by it, and the Adam update that takes the clipping factor along.
//
//   norm = sqrt(sum over all tensors and elements of g^2) / loss scale
//   c    = min(1, max_norm / (norm + 1e-6))           (a NaN norm gives a NaN factor, an infinite one the factor 0)
//   clip:  g <- c g          Adam:  g' = c g / loss scale + wd p, then the usual moments and update
//
// All of it streams memory: the norm reads every byte once, clipping reads again and writes, the update reads p, g,
// m, v (, vmax) and writes all but g.  Squares and sums are held in fp64: one conversion and one fp64 FMA per value
// are far below what the vector units can do while the value arrives from HBM, no square over- or underflows for any
// fp32 gradient (so the sum is finite exactly when every gradient is, which the loss scaler's overflow test uses),
// and the result is the exact sum to fp64 rounding.  No atomics: a list is cut into chunks, every chunk's sum goes to
// its own workspace slot and the slots are added in a fixed order, so equal inputs give equal bits.
//
// The tensor table travels in the kernel arguments (TABLE tensors a launch), so nothing has to be uploaded, kept alive
// or invalidated, and a captured launch carries its own copy.
#include "common.h"

namespace {

constexpr int TABLE = 160;            // tensors a launch: 160 x 21 bytes of kernel arguments, under the 4 KB limit
constexpr int THR = 256;
constexpr int MAX_CHUNKS = 2048;      // chunks a list is cut into, not counting each tensor's last one: 8 workgroups a CU
constexpr long long MIN_CHUNK = 16384;   // bytes: four 16-byte loads a thread
constexpr int FUSED_PARTS = 256;         // partial sums up to which the Adam update adds them up itself: one a thread.
                                         // 1 M values 10.8 us, with a launch of its own for that 11.5; 25 M (1500
                                         // sums, read by 6000 workgroups): 140 and 136
// Partial sums up to which every workgroup of the clipping launch adds them up itself: as many as a list has whose
// tensors are few.  Every tensor brings at least one more, so for long lists the sums would be quadratic work.  us, each
// workgroup / a launch of its own, norm included:
//   246 tensors, 1968 sums, 207 MB   49.3 / 49.7
//   tensors of 500 values            1000: 41.2 / 40.4   3000: 116 / 95   10000: 553 / 300   20000: 1732 / 728
constexpr int CLIP_PARTS = MAX_CHUNKS;
constexpr int SMALL_WAVES = 16;
constexpr long long SMALL_CHUNK = 4096;  // bytes a wave takes at a time in the single-workgroup form
// Chunks up to which one workgroup does everything; us, one workgroup and two launches, norm: 64 KB 3.2 / 4.6, 128 KB
// 4.2 / 4.5, 256 KB 6.4 / 4.7; clipping: 64 KB 5.7 / 6.7, 96 KB 6.6 / 6.8, 128 KB 8.5 / 6.8.
constexpr int SMALL_NORM = 32, SMALL_CLIP = 24;

struct Table {
  const void* p[TABLE];
  long long n[TABLE];                 // elements
  int first[TABLE];                   // first chunk of tensor i
  unsigned char type[TABLE];
  int count, chunks, part0;           // tensors, chunks of this launch, workspace slot of its first chunk
  long long chunk;                    // bytes a chunk
};

// The tensor that holds chunk b: the last one with first <= b (empty tensors are not in the table, so no two share a
// `first`).  One load a lane instead of a search.
__device__ __forceinline__ int tensor_of(const Table& t, int b) {
  const int lane = threadIdx.x & 63;
  int k = 0;
#pragma unroll
  for (int j = 0; j < (TABLE + 63) / 64; ++j) {
    const int i = j * 64 + lane;
    const bool le = i < t.count && t.first[i < TABLE ? i : 0] <= b;
    k += __popcll(__ballot(le));
  }
  return __builtin_amdgcn_readfirstlane(k - 1);
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T> union Piece {
  u32x4 u;
  T e[16 / sizeof(T)];
};

// The part of one chunk that lies in 16-byte pieces, and the elements before the tensor's first and behind its last
// whole piece.  Offsets are bytes from the tensor's start rounded down to 16, so every piece is aligned whatever the
// tensor's own alignment, and no byte outside the tensor is touched.
struct Span {
  long long v0, v1;                   // pieces [v0, v1)
  long long h0, h1, t0, t1;           // single elements [h0, h1) and [t0, t1), as byte offsets
};

__device__ __forceinline__ Span span_of(const void* p, long long n, int esz, long long c, long long chunk) {
  const long long beg = (long long)(reinterpret_cast<uintptr_t>(p) & 15), end = beg + n * esz;
  const long long lo = c * chunk, hi = min(lo + chunk, end);
  long long vf = (beg + 15) >> 4, vl = end >> 4;    // the tensor's whole pieces
  Span s;
  s.h0 = s.h1 = s.t0 = s.t1 = 0;
  if (vf > vl) {                      // the tensor lies inside one piece
    s.v0 = s.v1 = 0;
    s.h0 = beg;
    s.h1 = end;
    return s;
  }
  s.v0 = max(vf, lo >> 4);
  s.v1 = min(vl, (lo + chunk) >> 4);
  if (c == 0 && beg) {
    s.h0 = beg;
    s.h1 = vf << 4;
  }
  if (hi == end && (end & 15)) {
    s.t0 = vl << 4;
    s.t1 = end;
  }
  return s;
}

// Streaming accesses: what is read or written for the last time leaves no copy in the caches.  In front of a second
// pass they keep the first one's bytes in the 256 MB memory-side cache: clipping 52 M fp32 values 142 -> 119 us (read
// and written; read alone it stays at 144), the Adam update 404 -> 339 us; a norm alone, 2 GB of bf16, 335 -> 314 us.
__device__ __forceinline__ u32x4 load_once(const void* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
}

__device__ __forceinline__ void store_once(void* p, const u32x4& v) {
  __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p));
}

template <typename T, int NT, bool ONCE>
__device__ __forceinline__ double sumsq(const void* p, long long n, long long c, long long chunk, int tid) {
  const char* base = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)15);
  const Span s = span_of(p, n, sizeof(T), c, chunk);
  constexpr int N = 16 / (int)sizeof(T);
  double a0 = 0., a1 = 0.;
  auto add = [&](const u32x4& u) {
    Piece<T> q;
    q.u = u;
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const double x = (double)(float)q.e[e], y = (double)(float)q.e[e + 1];
      a0 = fma(x, x, a0);
      a1 = fma(y, y, a1);
    }
  };
  const u32x4* v = reinterpret_cast<const u32x4*>(base);
  auto load = [&](long long k) { return ONCE ? load_once(v + k) : v[k]; };
  long long i = s.v0 + tid;
  for (; i + 3 * NT < s.v1; i += 4 * NT) {          // four pieces in flight a thread
    const u32x4 u0 = load(i), u1 = load(i + NT), u2 = load(i + 2 * NT), u3 = load(i + 3 * NT);
    add(u0);
    add(u1);
    add(u2);
    add(u3);
  }
  for (; i < s.v1; i += NT) add(load(i));
  auto single = [&](long long b, long long e) {
    const long long o = b + (long long)tid * sizeof(T);
    if (o < e) {
      const double x = (double)(float)*reinterpret_cast<const T*>(base + o);
      a0 = fma(x, x, a0);
    }
  };
  single(s.h0, s.h1);                 // at most 15 elements: fewer than the threads
  single(s.t0, s.t1);
  return a0 + a1;
}

template <typename T, int NT>
__device__ __forceinline__ void scale_by(void* p, long long n, long long c, long long chunk, int tid, float f) {
  char* base = reinterpret_cast<char*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)15);
  const Span s = span_of(p, n, sizeof(T), c, chunk);
  constexpr int N = 16 / (int)sizeof(T);
  auto mul = [&](const u32x4& u) {
    Piece<T> q;
    q.u = u;
#pragma unroll
    for (int e = 0; e < N; ++e) q.e[e] = (T)((float)q.e[e] * f);
    return q.u;
  };
  u32x4* v = reinterpret_cast<u32x4*>(base);
  long long i = s.v0 + tid;
  for (; i + 3 * NT < s.v1; i += 4 * NT) {
    const u32x4 u0 = load_once(v + i), u1 = load_once(v + i + NT), u2 = load_once(v + i + 2 * NT),
                u3 = load_once(v + i + 3 * NT);
    store_once(v + i, mul(u0));
    store_once(v + i + NT, mul(u1));
    store_once(v + i + 2 * NT, mul(u2));
    store_once(v + i + 3 * NT, mul(u3));
  }
  for (; i < s.v1; i += NT) store_once(v + i, mul(load_once(v + i)));
  auto single = [&](long long b, long long e) {
    const long long o = b + (long long)tid * sizeof(T);
    if (o < e) {
      T* q = reinterpret_cast<T*>(base + o);
      *q = (T)((float)*q * f);
    }
  };
  single(s.h0, s.h1);
  single(s.t0, s.t1);
}

template <int NT, bool ONCE>
__device__ __forceinline__ double chunk_sumsq(const Table& t, int b, int tid) {
  const int k = tensor_of(t, b);
  const int c = b - t.first[k];
  if (t.type[k] == VCA_T_F32) return sumsq<float, NT, ONCE>(t.p[k], t.n[k], c, t.chunk, tid);
  if (t.type[k] == VCA_T_BF16) return sumsq<__bf16, NT, ONCE>(t.p[k], t.n[k], c, t.chunk, tid);
  return sumsq<_Float16, NT, ONCE>(t.p[k], t.n[k], c, t.chunk, tid);
}

template <int NT>
__device__ __forceinline__ void chunk_scale(const Table& t, int b, int tid, float f) {
  const int k = tensor_of(t, b);
  const int c = b - t.first[k];
  void* p = const_cast<void*>(t.p[k]);
  if (t.type[k] == VCA_T_F32) scale_by<float, NT>(p, t.n[k], c, t.chunk, tid, f);
  else if (t.type[k] == VCA_T_BF16) scale_by<__bf16, NT>(p, t.n[k], c, t.chunk, tid, f);
  else scale_by<_Float16, NT>(p, t.n[k], c, t.chunk, tid, f);
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Sum over a workgroup of NW waves, in every thread; the same order of additions in every workgroup.
template <int NW>
__device__ __forceinline__ double block_sum_d(double v, double* part) {
  v = wave_sum_d(v);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0.;
#pragma unroll
  for (int i = 0; i < NW; ++i) t += part[i];
  return t;
}

// norm and clipping factor from the sum of squares of the gradients as stored (scale: {s, 1/s} or null)
__device__ __forceinline__ double true_norm(double total, const float* scale) {
  return sqrt(total) * (scale ? (double)scale[1] : 1.);
}

__device__ __forceinline__ float clip_factor(double norm, float max_norm) {
  const double c = (double)max_norm / (norm + 1e-6);
  return c >= 1. ? 1.f : (float)c;    // a NaN stays one
}

// Partial sums, a chunk a workgroup.  Bound by memory: 2 GB of bf16 in 310 us, 6.4 TB/s; 207 MB of fp32 whose first
// part is still cached 39 us, 5.3 TB/s.
//   ONCE         nothing reads the tensors again behind it
//   step / next  where given, *next = *step + 1 on the way (see adam_clip_kernel)
template <bool ONCE>
__global__ __launch_bounds__(THR) void norm_chunks_kernel(const Table t, double* __restrict__ ws,
                                                          const int* __restrict__ step, int* __restrict__ next) {
  __shared__ double part[THR / 64];
  if (next && t.part0 + (int)blockIdx.x + (int)threadIdx.x == 0) *next = *step + 1;
  const double v = block_sum_d<THR / 64>(chunk_sumsq<THR, ONCE>(t, blockIdx.x, threadIdx.x), part);
  if (threadIdx.x == 0) ws[t.part0 + blockIdx.x] = v;
}

__device__ __forceinline__ double fold(const double* __restrict__ ws, int n, double* part) {
  double a = 0.;
  for (int i = threadIdx.x; i < n; i += THR) a += ws[i];
  return block_sum_d<THR / 64>(a, part);
}

__global__ __launch_bounds__(THR) void norm_fold_kernel(const double* __restrict__ ws, int n,
                                                        const float* __restrict__ scale, float* __restrict__ out) {
  __shared__ double part[THR / 64];
  const double total = fold(ws, n, part);
  if (threadIdx.x == 0) out[0] = (float)true_norm(total, scale);
}

// The sum of a long list's slots into the first of them: all have been read behind the sum's barrier.
__global__ __launch_bounds__(THR) void norm_total_kernel(double* __restrict__ ws, int n) {
  __shared__ double part[THR / 64];
  const double total = fold(ws, n, part);
  if (threadIdx.x == 0) ws[0] = total;
}

// Every workgroup adds up the slots itself (out of L2, under the time of one more launch; n is 1 for a list whose
// tensors are so many that norm_total_kernel has done it, CLIP_PARTS) and scales its chunk; with a factor of one
// there is nothing to do.  Chunks are taken from the last to the first: the norm's pass left the end of the list in
// the caches (400 MB 192 us, from the first 200).  Bound by memory: norm and clipping of 207 MB together 119 us, 5.2
// TB/s of the 621 MB read and written.
__global__ __launch_bounds__(THR) void clip_chunks_kernel(const Table t, const double* __restrict__ ws, int n,
                                                          float max_norm, const float* __restrict__ scale,
                                                          float* __restrict__ out) {
  __shared__ double part[THR / 64];
  const double norm = true_norm(fold(ws, n, part), scale);
  if (out && blockIdx.x == 0 && threadIdx.x == 0) out[0] = (float)norm;
  const float f = clip_factor(norm, max_norm);
  if (f == 1.f) return;
  chunk_scale<THR>(t, t.chunks - 1 - (int)blockIdx.x, threadIdx.x, f);
}

// Short lists: one workgroup whose waves take chunks in turn, so that norm and clipping are a single launch.
template <bool CLIP>
__global__ __launch_bounds__(SMALL_WAVES * 64) void norm_small_kernel(const Table t, float max_norm,
                                                                      const float* __restrict__ scale,
                                                                      float* __restrict__ out) {
  __shared__ double part[SMALL_WAVES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  double a = 0.;
  for (int b = wave; b < t.chunks; b += SMALL_WAVES) a += chunk_sumsq<64, false>(t, b, lane);
  const double norm = true_norm(block_sum_d<SMALL_WAVES>(a, part), scale);
  if (threadIdx.x == 0) out[0] = (float)norm;
  if (!CLIP) return;
  const float f = clip_factor(norm, max_norm);
  if (f == 1.f) return;
  for (int b = wave; b < t.chunks; b += SMALL_WAVES) chunk_scale<64>(t, b, lane, f);
}

// ---------------------------------------------------------------------------------------------------------------
// Adam with the clipping factor
// ---------------------------------------------------------------------------------------------------------------
struct Groups {
  vca_adam_group g[VCA_MAX_ADAM_GROUPS];
  int first[VCA_MAX_ADAM_GROUPS];     // first workgroup of group i
  int count;
  long long chunk4;                   // float4s a workgroup
};

struct AdamCfg {
  float b1, b2, omb1, omb2, eps, wd;  // omb = 1 - beta, rounded once (1.f - 0.999f is off by 1e-5 of itself)
  double b1d, b2d;
};

// The step's words from the sum of squares, by one thread:
// {norm, c / loss scale, learning rate / (1 - b1^t), sqrt(1 - b2^t)}.  Returns whether there is a step: with a scaler a gradient that is not finite raises the flag, and the
// count stays.  `step` is this step's number.
struct AdamWords { float norm, factor, rate, root; };

__device__ __forceinline__ bool adam_words(double total, float max_norm, const float* scale, const int* flag, int step,
                                           const float* lr_dev, const AdamCfg& cfg, AdamWords& w) {
  const double norm = true_norm(total, scale);
  w.norm = (float)norm;
  w.factor = clip_factor(norm, max_norm) * (scale ? scale[1] : 1.f);
  const double t = (double)step;
  w.rate = (float)((double)lr_dev[0] / (1. - pow(cfg.b1d, t)));
  w.root = (float)sqrt(1. - pow(cfg.b2d, t));
  return !flag || (flag[0] == 0 && isfinite(total));
}

struct AdamArgs {
  const double* ws;                   // partial sums of squares
  int parts;
  float max_norm;
  const float* scale;
  int* flag;
  int* step_dev;
  const float* lr_dev;
  float* out;                         // AdamWords, and the step's number as an int behind them
};

__device__ __forceinline__ void publish(const AdamArgs& a, const AdamWords& w, bool go, double total, int step) {
  a.out[0] = w.norm;
  a.out[1] = w.factor;
  a.out[2] = w.rate;
  a.out[3] = w.root;
  if (go) a.step_dev[0] = step;
  else if (!isfinite(total)) a.flag[0] = 1;
}

__global__ __launch_bounds__(THR) void adam_words_kernel(const AdamArgs a, const AdamCfg cfg) {
  __shared__ double part[THR / 64];
  const double total = fold(a.ws, a.parts, part);
  if (threadIdx.x) return;
  AdamWords w;
  const int step = a.step_dev[0] + 1;
  const bool go = adam_words(total, a.max_norm, a.scale, a.flag, step, a.lr_dev, cfg, w);
  publish(a, w, go, total, step);
}

union Four {
  u32x4 u;
  float f[4];
};

__device__ __forceinline__ void adam4(float (&p)[4], const float (&g)[4], float (&m)[4], float (&v)[4], float (&x)[4],
                                      bool ams, const AdamCfg& c, float f, float step, float root) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float gr = g[j] * f + c.wd * p[j];
    m[j] = c.b1 * m[j] + c.omb1 * gr;
    v[j] = c.b2 * v[j] + c.omb2 * gr * gr;
    float q = v[j];
    if (ams) q = x[j] = fmaxf(x[j], v[j]);
    p[j] -= step * m[j] / (sqrtf(q) / root + c.eps);
  }
}

// FUSED (few partial sums): every workgroup adds the sums up and forms the words itself, which saves the launch in
// between (FUSED_PARTS).  The step's number then comes from out[4], where the norm's launch
// left it: the first workgroup writes the new count while others may still be starting.
// Bound by memory: 52 M values with amsgrad (36 bytes each, some of it cached by the norm's pass) 304 us, 6.1 TB/s.
template <bool FUSED>
__global__ __launch_bounds__(THR) void adam_clip_kernel(const Groups t, const AdamCfg cfg, const AdamArgs a) {
  __shared__ double part[THR / 64];
  __shared__ AdamWords sw;
  __shared__ bool sgo;
  if (FUSED) {
    const double total = fold(a.ws, a.parts, part);
    if (threadIdx.x == 0) {
      const int step = reinterpret_cast<const int*>(a.out)[4];
      AdamWords w;
      const bool go = adam_words(total, a.max_norm, a.scale, a.flag, step, a.lr_dev, cfg, w);
      sw = w;
      sgo = go;
      if (blockIdx.x == 0) publish(a, w, go, total, step);
    }
    __syncthreads();
    if (!sgo) return;
  } else if (a.flag && a.flag[0]) {
    return;
  }
  int k = 0;
  for (int i = 1; i < t.count; ++i)
    if (t.first[i] <= (int)blockIdx.x) k = i;
  const vca_adam_group g = t.g[k];
  const float f = FUSED ? sw.factor : a.out[1], step = FUSED ? sw.rate : a.out[2], root = FUSED ? sw.root : a.out[3];
  const bool ams = g.vmax != nullptr;
  const long long n4 = g.n >> 2, lo = (long long)(blockIdx.x - t.first[k]) * t.chunk4, hi = min(lo + t.chunk4, n4);
  float4 *p = reinterpret_cast<float4*>(g.p), *m = reinterpret_cast<float4*>(g.m), *v = reinterpret_cast<float4*>(g.v),
         *x = reinterpret_cast<float4*>(g.vmax);
  const float4* gr = reinterpret_cast<const float4*>(g.g);
  for (long long i = lo + threadIdx.x; i < hi; i += THR) {
    Four P, M, V, X, G;
    P.u = load_once(p + i);
    M.u = load_once(m + i);
    V.u = load_once(v + i);
    G.u = load_once(gr + i);
    if (ams) X.u = load_once(x + i);
    adam4(P.f, G.f, M.f, V.f, X.f, ams, cfg, f, step, root);
    store_once(p + i, P.u);
    store_once(m + i, M.u);
    store_once(v + i, V.u);
    if (ams) store_once(x + i, X.u);
  }
}

int type_size(int t) { return t == VCA_T_F32 ? 4 : (t == VCA_T_BF16 || t == VCA_T_F16) ? 2 : 0; }

// Checks a list and finds its bytes; false for one that no kernel may see.
bool list_ok(int n, const void* const* p, const long long* numel, const int* type, long long& bytes) {
  if (n < 0 || (n && (!p || !numel || !type))) return false;
  bytes = 0;
  for (int i = 0; i < n; ++i) {
    const int e = type_size(type[i]);
    if (!e || numel[i] < 0 || numel[i] > (1ll << 46)) return false;
    if (numel[i] && (!p[i] || (reinterpret_cast<uintptr_t>(p[i]) & (e - 1)))) return false;
    bytes += numel[i] * e;
  }
  return true;
}

long long chunks_of(const void* p, long long numel, int e, long long chunk) {
  if (!numel) return 0;
  return ((long long)(reinterpret_cast<uintptr_t>(p) & 15) + numel * e + chunk - 1) / chunk;
}

long long chunk_bytes(long long bytes) {
  const long long c = (bytes / MAX_CHUNKS + MIN_CHUNK - 1) / MIN_CHUNK * MIN_CHUNK;
  return c < MIN_CHUNK ? MIN_CHUNK : c;
}

// Fills a launch's table with the list's tensors from i on (empty ones are left out); returns the next tensor.
int fill(Table& t, int i, int n, const void* const* p, const long long* numel, const int* type, long long chunk,
         int part0) {
  t.count = t.chunks = 0;
  t.part0 = part0;
  t.chunk = chunk;
  for (; i < n && t.count < TABLE; ++i) {
    const long long c = chunks_of(p[i], numel[i], type_size(type[i]), chunk);
    if (!c) continue;
    t.p[t.count] = p[i];
    t.n[t.count] = numel[i];
    t.type[t.count] = (unsigned char)type[i];
    t.first[t.count] = t.chunks;
    t.chunks += (int)c;
    ++t.count;
  }
  return i;
}

long long total_chunks(int n, const void* const* p, const long long* numel, const int* type, long long chunk) {
  long long c = 0;
  for (int i = 0; i < n; ++i) c += chunks_of(p[i], numel[i], type_size(type[i]), chunk);
  return c;
}

// Launches the partial sums of a list; parts = slots written.
int norm_partials(bool once, int n, const void* const* p, const long long* numel, const int* type, long long bytes, double* ws,
                  long long ws_doubles, hipStream_t s, int& parts, const int* step = nullptr, int* next = nullptr) {
  const long long chunk = chunk_bytes(bytes);
  const long long need = total_chunks(n, p, numel, type, chunk);
  VCA_CHECK_ARG(need <= ws_doubles && (need == 0 || (ws && (reinterpret_cast<uintptr_t>(ws) & 7) == 0)));
  parts = 0;
  Table t;
  for (int i = 0; i < n;) {
    i = fill(t, i, n, p, numel, type, chunk, parts);
    if (t.chunks && once) hipLaunchKernelGGL(norm_chunks_kernel<true>, dim3(t.chunks), dim3(THR), 0, s, t, ws, step, next);
    if (t.chunks && !once) hipLaunchKernelGGL(norm_chunks_kernel<false>, dim3(t.chunks), dim3(THR), 0, s, t, ws, step, next);
    parts += t.chunks;
  }
  return vca_launch_status();
}

// One workgroup is enough: the whole list in one table and few chunks.
bool small_list(int n, const void* const* p, const long long* numel, const int* type, int items, Table& t) {
  if (total_chunks(n, p, numel, type, SMALL_CHUNK) > items) return false;
  return fill(t, 0, n, p, numel, type, SMALL_CHUNK, 0) == n;
}

}  // namespace

extern "C" long long vca_grad_norm_ws_doubles(int ntensor, const void* const* h_ptrs, const long long* h_numel,
                                              const int* h_types) {
  long long bytes = 0;
  if (ntensor < 0) return 0;
  if (!h_ptrs) return MAX_CHUNKS + 2ll * ntensor;
  if (!list_ok(ntensor, h_ptrs, h_numel, h_types, bytes)) return 0;
  Table t;
  if (small_list(ntensor, h_ptrs, h_numel, h_types, SMALL_CLIP, t)) return 0;   // (the smaller of the two)
  return total_chunks(ntensor, h_ptrs, h_numel, h_types, chunk_bytes(bytes));
}

extern "C" int vca_grad_norm(int ntensor, const void* const* h_ptrs, const long long* h_numel, const int* h_types,
                             const float* scale, double* ws, long long ws_doubles, float* out, void* stream) {
  long long bytes = 0;
  VCA_CHECK_ARG(out && list_ok(ntensor, h_ptrs, h_numel, h_types, bytes));
  hipStream_t s = (hipStream_t)stream;
  Table t;
  if (small_list(ntensor, h_ptrs, h_numel, h_types, SMALL_NORM, t)) {
    hipLaunchKernelGGL(norm_small_kernel<false>, dim3(1), dim3(SMALL_WAVES * 64), 0, s, t, 0.f, scale, out);
    return vca_launch_status();
  }
  int parts = 0;
  const int rc = norm_partials(true, ntensor, h_ptrs, h_numel, h_types, bytes, ws, ws_doubles, s, parts);
  if (rc) return rc;
  hipLaunchKernelGGL(norm_fold_kernel, dim3(1), dim3(THR), 0, s, ws, parts, scale, out);
  return vca_launch_status();
}

extern "C" int vca_grad_clip(int ntensor, const void* const* h_ptrs, const long long* h_numel, const int* h_types,
                             float max_norm, const float* scale, double* ws, long long ws_doubles, float* out,
                             void* stream) {
  long long bytes = 0;
  VCA_CHECK_ARG(out && max_norm >= 0.f && list_ok(ntensor, h_ptrs, h_numel, h_types, bytes));
  hipStream_t s = (hipStream_t)stream;
  Table t;
  if (small_list(ntensor, h_ptrs, h_numel, h_types, SMALL_CLIP, t)) {
    hipLaunchKernelGGL(norm_small_kernel<true>, dim3(1), dim3(SMALL_WAVES * 64), 0, s, t, max_norm, scale, out);
    return vca_launch_status();
  }
  int parts = 0;
  const int rc = norm_partials(false, ntensor, h_ptrs, h_numel, h_types, bytes, ws, ws_doubles, s, parts);
  if (rc) return rc;
  if (parts > CLIP_PARTS) {
    hipLaunchKernelGGL(norm_total_kernel, dim3(1), dim3(THR), 0, s, ws, parts);
    parts = 1;
  }
  const long long chunk = chunk_bytes(bytes);
  bool first = true;
  for (int end = ntensor; end > 0;) {                    // tables from the end of the list backwards
    int beg = end, used = 0;
    while (beg > 0 && used < TABLE) used += h_numel[--beg] > 0;
    fill(t, beg, end, h_ptrs, h_numel, h_types, chunk, 0);
    end = beg;
    if (!t.chunks) continue;
    hipLaunchKernelGGL(clip_chunks_kernel, dim3(t.chunks), dim3(THR), 0, s, t, ws, parts, max_norm, scale,
                       first ? out : nullptr);
    first = false;
  }
  return vca_launch_status();
}

extern "C" int vca_adam_clip_f32(int ngroup, const vca_adam_group* h_groups, float max_norm, double beta1, double beta2,
                                 double eps, double weight_decay, int* step_dev, const float* lr_dev,
                                 const float* scale, int* flag, double* ws, long long ws_doubles, float* out,
                                 void* stream) {
  VCA_CHECK_ARG(ngroup >= 1 && ngroup <= VCA_MAX_ADAM_GROUPS && h_groups && max_norm >= 0.f && step_dev && lr_dev && out);
  VCA_CHECK_ARG(!scale == !flag);
  const void* p[VCA_MAX_ADAM_GROUPS];
  long long numel[VCA_MAX_ADAM_GROUPS], total = 0;
  int type[VCA_MAX_ADAM_GROUPS];
  Groups t;
  t.count = ngroup;
  for (int i = 0; i < ngroup; ++i) {
    const vca_adam_group& g = h_groups[i];
    VCA_CHECK_ARG(g.n > 0 && (g.n % 4) == 0 && g.n <= (1ll << 44) && g.p && g.g && g.m && g.v);
    VCA_CHECK_ARG(((reinterpret_cast<uintptr_t>(g.p) | reinterpret_cast<uintptr_t>(g.g) | reinterpret_cast<uintptr_t>(g.m) |
                    reinterpret_cast<uintptr_t>(g.v) | reinterpret_cast<uintptr_t>(g.vmax)) & 15) == 0);
    p[i] = g.g;
    numel[i] = g.n;
    type[i] = VCA_T_F32;
    t.g[i] = g;
    total += g.n;
  }
  hipStream_t s = (hipStream_t)stream;
  int parts = 0;
  const int rc = norm_partials(false, ngroup, p, numel, type, total * 4, ws, ws_doubles, s, parts, step_dev,
                               reinterpret_cast<int*>(out) + 4);
  if (rc) return rc;
  AdamCfg cfg;
  cfg.b1 = (float)beta1;
  cfg.b2 = (float)beta2;
  cfg.omb1 = (float)(1. - beta1);
  cfg.omb2 = (float)(1. - beta2);
  cfg.eps = (float)eps;
  cfg.wd = (float)weight_decay;
  cfg.b1d = beta1;
  cfg.b2d = beta2;
  const AdamArgs args = {ws, parts, max_norm, scale, flag, step_dev, lr_dev, out};
  const bool fused = parts <= FUSED_PARTS;
  if (!fused) hipLaunchKernelGGL(adam_words_kernel, dim3(1), dim3(THR), 0, s, args, cfg);
  // 4 float4s a thread, more where the list is so long that this would be over 16384 workgroups
  t.chunk4 = 4 * THR;
  while ((total / 4) / t.chunk4 > 16384) t.chunk4 *= 2;
  int blocks = 0;
  for (int i = 0; i < ngroup; ++i) {
    t.first[i] = blocks;
    blocks += (int)((numel[i] / 4 + t.chunk4 - 1) / t.chunk4);
  }
  if (fused) hipLaunchKernelGGL(adam_clip_kernel<true>, dim3(blocks), dim3(THR), 0, s, t, cfg, args);
  else hipLaunchKernelGGL(adam_clip_kernel<false>, dim3(blocks), dim3(THR), 0, s, t, cfg, args);
  return vca_launch_status();
}
