// seq_norm.hip — the residual's addition with the root-mean-square norm, its 8-bit output, its
// gradient, and rows quantised to 8 bits (include/pnp.h pnp_rms_norm, pnp_rms_norm_bwd,
// pnp_quantize_rows).
//
//   s = x + r (rounded to the stream's type: what later layers read is what is normalised),
//   rho = 1 / sqrt(mean(s^2) + eps), n = s rho, y = n w
//   dx = ds + rho (w dy - n mean(w dy n)),  dw = sum over rows of dy n
//
// Bound by HBM: a row is read once, kept in registers between its sums and its outputs, and written
// once.  A row that fits gets 8, 16 or 32 lanes with a pack each, a longer one a wave (up to 4 packs a
// lane), then a workgroup of 256 threads (up to 8 packs a thread); rows past that are read twice (the
// second time from cache).
//
// Rows that are no whole packs, or not on their boundaries (EVEN false): packs from wherever they lie,
// the last one moved back to end with the row.  Its first elements are another lane's too: written
// twice, the same value, and counted once.
//
// Measured, with a residual: bf16, 8192 x 4096, 42 us forward (268 MB, 6.3 TB/s: part of it from cache), 63 back with
// the weight's sums (336 MB); 16384 x 4096 both in 210 us (1.07 GB at 5.1 TB/s, a large copy's rate); rows of 4095 45
// and 89 us, of 4100 54 and 100 (by elements, of 4095, 96 and 167); 200000 rows of 64 19 and 23 us (by whole waves 61
// forward).
#include <type_traits>

#include "seq_dev.h"

namespace seq {
namespace {

constexpr int NT = 256;

struct NormArgs {
  int64_t rows, xs, rs, qs;
  int dim;
  float eps;
  const void *x, *r;
  const float* w;
  void *y, *s;
  float* rstd;
  int8_t* q;
  float* scale;
};

// sum over the TPR threads of a row, in each of them; red: NT / 64 floats of LDS, a use apart each call
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* red) {
  v = group_sum<TPR < 64 ? TPR : 64>(v);
  if (TPR <= 64) return v;
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) red[w] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}
template <int TPR> __device__ __forceinline__ float row_max(float v, float* red) {
  v = group_max_nan<TPR < 64 ? TPR : 64>(v);
  if (TPR <= 64) return v;
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) red[w] = v;
  __syncthreads();
  return max_nan(max_nan(red[0], red[1]), max_nan(red[2], red[3]));
}

// a lane's pack of a row: where it lies, and how many of its elements are its neighbour's
template <int V, bool EVEN> struct Place {
  int i, skip;
  bool on;
  __device__ __forceinline__ Place(int at, int dim) : i(at), skip(0), on(at < dim) {
    if (!EVEN && at + V > dim) {
      skip = at + V - dim;
      i = dim - V;
    }
  }
  __device__ __forceinline__ bool own(int k) const { return EVEN || k >= skip; }
  __device__ __forceinline__ float once(int k, float v) const { return own(k) ? v : 0.f; }   // v where the element counts
};

// What a row whose largest magnitude is m is scaled by: scale = m / 127, 0 where that would be below the least normal
// number, NaN where m is not finite.  by and inv: scale and 1 / scale, of values times lift (2^64 in rows of less than
// 2^-60, so that the remainder below does not fall under fp32; 1 otherwise); inv = 0 where scale is 0 or NaN.
struct Steps {
  float scale, by, inv, lift;
  __device__ __forceinline__ explicit Steps(float m) : scale(m / 127.f) {
    lift = scale < 0x1p-60f ? 0x1p64f : 1.f;
    by = scale * lift;
    inv = 1.f / by;
    if (!(m < __builtin_inff())) { scale = __builtin_nanf(""); inv = 0.f; }
    else if (scale < 0x1p-126f) { scale = 0.f; inv = 0.f; }
  }
};
// q = the fp32 quotient y / scale, rounded to nearest even.  The product y inv is up to 1.5 steps of fp32 off it, which
// shows next to the halves between two of q; with its remainder's share added none of them is missed (all 2^23
// mantissas of scale times all halves times the 16 values of y next to each, counted).  Rows in 8 bits, bf16, 8192 x 1024:
// 6.7 us, by the product alone 6.6, with a division for the packs that come near a half 8.5.
// inv = 0 gives q = 0 for the finite values of a row; NaN (of infinity too) becomes 0 here.
template <int V, bool EVEN> __device__ __forceinline__ void store_q8(int8_t* p, const float (&y)[V], const Steps& s) {
  typename PackOf<int8_t, V, EVEN>::type o;
#pragma unroll
  for (int k = 0; k < V; k++) {
    const float l = y[k] * s.lift, v = l * s.inv, r = rintf(fmaf(fmaf(-v, s.by, l), s.inv, v));
    o.v[k] = (int8_t)(int)(r == r ? r : 0.f);
  }
  *reinterpret_cast<typename PackOf<int8_t, V, EVEN>::type*>(p) = o;
}

// T: x and y; R: the residual stream; V elements a load; TPR threads a row; NV packs a thread (0: rows
// of any length, read twice); Q8: 8-bit output
template <typename T, typename R, int V, bool EVEN, int TPR, int NV, bool Q8>
__device__ __forceinline__ void norm_fwd_row(const NormArgs& a, int64_t row, float (&red)[2][NT / 64]) {
  typedef Place<V, EVEN> At;
  const int lane = threadIdx.x % TPR;
  const T* x = (const T*)a.x + row * a.xs;
  const R* r = a.r ? (const R*)a.r + row * a.rs : nullptr;
  R* so = a.s ? (R*)a.s + row * a.dim : nullptr;
  auto read = [&](int i, float (&v)[V]) {
    load_f<V, EVEN>(x + i, v);
    if (r) {
      float b[V];
      load_f<V, EVEN>(r + i, b);
#pragma unroll
      for (int k = 0; k < V; k++) v[k] = to_f(from_f<R>(v[k] + b[k]));
    }
  };
  // short rows take their weights along with the row, not after its sum
  constexpr bool EARLY = NV == 1;
  float early[V];
  if (EARLY && a.w && lane * V < a.dim) load_f<V, EVEN>(a.w + At(lane * V, a.dim).i, early);
  auto scaled = [&](int i, float rho, float (&v)[V]) {
    float w[V];
    if (EARLY)
#pragma unroll
      for (int k = 0; k < V; k++) w[k] = early[k];
    else if (a.w) load_f<V, EVEN>(a.w + i, w);
#pragma unroll
    for (int k = 0; k < V; k++) v[k] = a.w ? v[k] * rho * w[k] : v[k] * rho;
  };
  float sum = 0.f, m = 0.f;
  if constexpr (NV > 0) {
    float v[NV][V];
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const At p((j * TPR + lane) * V, a.dim);
      if (p.on) read(p.i, v[j]);
      else
#pragma unroll
        for (int k = 0; k < V; k++) v[j][k] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const At p((j * TPR + lane) * V, a.dim);
      if (so && p.on) store_f<V, EVEN>(so + p.i, v[j]);
#pragma unroll
      for (int k = 0; k < V; k++) sum += p.once(k, v[j][k]) * p.once(k, v[j][k]);
    }
    const float rho = 1.f / sqrtf(row_sum<TPR>(sum, red[0]) / (float)a.dim + a.eps);
    if (a.rstd && lane == 0) a.rstd[row] = rho;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const At p((j * TPR + lane) * V, a.dim);
      if (!p.on) continue;
      scaled(p.i, rho, v[j]);
      if constexpr (Q8) {
#pragma unroll
        for (int k = 0; k < V; k++) m = max_nan(m, fabsf(v[j][k]));
      } else {
        store_f<V, EVEN>((T*)a.y + row * a.dim + p.i, v[j]);
      }
    }
    if constexpr (Q8) {
      const Steps by(row_max<TPR>(m, red[1]));
      if (lane == 0) a.scale[row] = by.scale;
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const At p((j * TPR + lane) * V, a.dim);
        if (!p.on) continue;
        store_q8<V, EVEN>(a.q + row * a.qs + p.i, v[j], by);
      }
    }
  } else {
    for (int c = lane * V; c < a.dim; c += TPR * V) {
      const At p(c, a.dim);
      float v[V];
      read(p.i, v);
      if (so) store_f<V, EVEN>(so + p.i, v);
#pragma unroll
      for (int k = 0; k < V; k++) sum += p.once(k, v[k]) * p.once(k, v[k]);
    }
    const float rho = 1.f / sqrtf(row_sum<TPR>(sum, red[0]) / (float)a.dim + a.eps);
    if (a.rstd && lane == 0) a.rstd[row] = rho;
    for (int c = lane * V; c < a.dim; c += TPR * V) {
      const At p(c, a.dim);
      float v[V];
      read(p.i, v);
      scaled(p.i, rho, v);
      if constexpr (Q8) {
#pragma unroll
        for (int k = 0; k < V; k++) m = max_nan(m, fabsf(v[k]));
      } else {
        store_f<V, EVEN>((T*)a.y + row * a.dim + p.i, v);
      }
    }
    if constexpr (Q8) {
      const Steps by(row_max<TPR>(m, red[1]));
      if (lane == 0) a.scale[row] = by.scale;
      for (int c = lane * V; c < a.dim; c += TPR * V) {
        const At p(c, a.dim);
        float v[V];
        read(p.i, v);
        scaled(p.i, rho, v);
        store_q8<V, EVEN>(a.q + row * a.qs + p.i, v, by);
      }
    }
  }
}

// rows dealt to the grid; up to a wave (TPR 64) or the whole workgroup works on one
#define SEQ_ROWS(BODY)                                                                                      \
  for (int64_t row = (int64_t)blockIdx.x * (NT / TPR) + threadIdx.x / TPR; row < a.rows;                    \
       row += (int64_t)gridDim.x * (NT / TPR)) {                                                            \
    BODY;                                                                                                   \
    if (TPR > 64) __syncthreads(); /* the next row's sums go where this row's were read */                  \
  }

template <typename T, typename R, int V, bool EVEN, int TPR, int NV, bool Q8>
__global__ __launch_bounds__(NT) void norm_fwd_kernel(NormArgs a) {
  __shared__ float red[2][NT / 64];
  SEQ_ROWS((norm_fwd_row<T, R, V, EVEN, TPR, NV, Q8>(a, row, red)))
}

// rows in 8 bits: the norm's kernel without the norm (bf16, 8192 x 1024: 6.7 us in a captured row of 20 such launches)
template <typename T, int V, bool EVEN, int TPR, int NV>
__device__ __forceinline__ void quantize_row(const NormArgs& a, int64_t row, float (&red)[NT / 64]) {
  typedef Place<V, EVEN> At;
  const int lane = threadIdx.x % TPR;
  const T* x = (const T*)a.x + row * a.xs;
  int8_t* q = a.q + row * a.qs;
  float m = 0.f;
  if constexpr (NV > 0) {
    float v[NV][V];
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const At p((j * TPR + lane) * V, a.dim);
#pragma unroll
      for (int k = 0; k < V; k++) v[j][k] = 0.f;
      if (p.on) load_f<V, EVEN>(x + p.i, v[j]);
#pragma unroll
      for (int k = 0; k < V; k++) m = max_nan(m, fabsf(v[j][k]));
    }
    const Steps by(row_max<TPR>(m, red));
    if (lane == 0) a.scale[row] = by.scale;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const At p((j * TPR + lane) * V, a.dim);
      if (!p.on) continue;
      store_q8<V, EVEN>(q + p.i, v[j], by);
    }
  } else {
    for (int c = lane * V; c < a.dim; c += TPR * V) {
      const At p(c, a.dim);
      float v[V];
      load_f<V, EVEN>(x + p.i, v);
#pragma unroll
      for (int k = 0; k < V; k++) m = max_nan(m, fabsf(v[k]));
    }
    const Steps by(row_max<TPR>(m, red));
    if (lane == 0) a.scale[row] = by.scale;
    for (int c = lane * V; c < a.dim; c += TPR * V) {
      const At p(c, a.dim);
      float v[V];
      load_f<V, EVEN>(x + p.i, v);
      store_q8<V, EVEN>(q + p.i, v, by);
    }
  }
}

template <typename T, int V, bool EVEN, int TPR, int NV> __global__ __launch_bounds__(NT) void quantize_kernel(NormArgs a) {
  __shared__ float red[NT / 64];
  SEQ_ROWS((quantize_row<T, V, EVEN, TPR, NV>(a, row, red)))
}

struct NormBwdArgs {
  int64_t rows, dys, dss, ss;
  int dim;
  const void *dy, *ds, *s;
  const float *w, *rstd;
  void *dx, *dres;
  float* part;   // [gridDim.x][dim] sums of dy n, or null
};

// A workgroup takes rows blockIdx, blockIdx + gridDim, ...: the weight's gradient stays in registers
// over all of them (a thread keeps its columns) and leaves as one row of `part`.
template <typename T, typename R, int V, bool EVEN, int TPR, int NV>
__global__ __launch_bounds__(NT) void norm_bwd_kernel(NormBwdArgs a) {
  typedef Place<V, EVEN> At;
  constexpr int RPB = NT / TPR;
  __shared__ float red[2][NT / 64];
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  float acc[NV > 0 ? NV : 1][V] = {};
  int flip = 0;
  const float rdim = 1.f / (float)a.dim;
  for (int64_t row = (int64_t)blockIdx.x * RPB + sub; row < a.rows; row += (int64_t)gridDim.x * RPB) {
    const T* dy = (const T*)a.dy + row * a.dys;
    const R* s = (const R*)a.s + row * a.ss;
    const R* ds = a.ds ? (const R*)a.ds + row * a.dss : nullptr;
    T* dx = (T*)a.dx + row * a.dim;
    R* dr = a.dres ? (R*)a.dres + row * a.dim : nullptr;
    const float rho = a.rstd[row];
    float dot = 0.f;
    auto pair = [&](int i, float (&g)[V], float (&n)[V]) {
      load_f<V, EVEN>(dy + i, g);
      load_f<V, EVEN>(s + i, n);
#pragma unroll
      for (int k = 0; k < V; k++) n[k] *= rho;
    };
    auto weigh = [&](int i, float (&g)[V]) {
      float w[V];
      if (!a.w) return;
      load_f<V, EVEN>(a.w + i, w);
#pragma unroll
      for (int k = 0; k < V; k++) g[k] *= w[k];
    };
    auto put = [&](int i, float mean, const float (&g)[V], const float (&n)[V]) {
      float d[V], b[V];
      if (ds) load_f<V, EVEN>(ds + i, b);
#pragma unroll
      for (int k = 0; k < V; k++) {
        d[k] = rho * (g[k] - n[k] * mean);
        if (ds) d[k] += b[k];
      }
      store_f<V, EVEN>(dx + i, d);
      if (dr) store_f<V, EVEN>(dr + i, d);
    };
    if constexpr (NV > 0) {
      float g[NV][V], n[NV][V];
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const At p((j * TPR + lane) * V, a.dim);
        if (p.on) pair(p.i, g[j], n[j]);
        else
#pragma unroll
          for (int k = 0; k < V; k++) g[j][k] = n[j][k] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const At p((j * TPR + lane) * V, a.dim);
        if (!p.on) continue;
#pragma unroll
        for (int k = 0; k < V; k++) acc[j][k] += g[j][k] * n[j][k];
        weigh(p.i, g[j]);
#pragma unroll
        for (int k = 0; k < V; k++) dot += p.once(k, g[j][k]) * p.once(k, n[j][k]);
      }
      const float mean = row_sum<TPR>(dot, red[flip]) * rdim;
      flip ^= 1;   // (the next row's sums may be written while a slow wave still reads this row's)
#pragma unroll
      for (int j = 0; j < NV; j++) {
        const At p((j * TPR + lane) * V, a.dim);
        if (p.on) put(p.i, mean, g[j], n[j]);
      }
    } else {
      for (int c = lane * V; c < a.dim; c += TPR * V) {
        const At p(c, a.dim);
        float g[V], n[V];
        pair(p.i, g, n);
        weigh(p.i, g);
#pragma unroll
        for (int k = 0; k < V; k++) dot += p.once(k, g[k]) * p.once(k, n[k]);
      }
      const float mean = row_sum<TPR>(dot, red[flip]) * rdim;
      flip ^= 1;
      for (int c = lane * V; c < a.dim; c += TPR * V) {
        const At p(c, a.dim);
        float g[V], n[V];
        pair(p.i, g, n);
        weigh(p.i, g);
        put(p.i, mean, g, n);
      }
    }
  }
  if constexpr (NV > 0) {
    if (!a.part) return;
    float* part = a.part + (int64_t)blockIdx.x * a.dim;
    auto leave = [&](const At& p, const float (&sums)[V]) {   // (a column's sum is its owner's)
#pragma unroll
      for (int k = 0; k < V; k++)
        if (p.on && p.own(k)) part[p.i + k] = sums[k];
    };
    if constexpr (RPB > 1) {   // the rows' sums of the same columns, in the order of their lanes
      __shared__ float sh[RPB - 1][TPR * V];
#pragma unroll
      for (int j = 0; j < NV; j++) {
        if (sub)
#pragma unroll
          for (int k = 0; k < V; k++) sh[sub - 1][lane * V + k] = acc[j][k];
        __syncthreads();
        if (!sub) {
#pragma unroll 4
          for (int u = 0; u < RPB - 1; u++)
#pragma unroll
            for (int k = 0; k < V; k++) acc[j][k] += sh[u][lane * V + k];
          leave(At((j * TPR + lane) * V, a.dim), acc[j]);
        }
        __syncthreads();
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; j++) leave(At((j * TPR + lane) * V, a.dim), acc[j]);
    }
  }
}

// sums of dy n over a strip of rows, a thread a column: for rows too wide for registers
template <typename T, typename R> __global__ __launch_bounds__(NT) void norm_dw_kernel(NormBwdArgs a) {
  const int c = blockIdx.x * NT + threadIdx.x;
  if (c >= a.dim) return;
  float acc = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y)
    acc += to_f(((const T*)a.dy)[row * a.dys + c]) * (to_f(((const R*)a.s)[row * a.ss + c]) * a.rstd[row]);
  a.part[(int64_t)blockIdx.y * a.dim + c] = acc;
}

// 64 columns a workgroup, the rows dealt to 16 waves, their sums joined in wave order
__global__ __launch_bounds__(1024) void column_sums_kernel(const float* part, int64_t n, int64_t stride, int64_t cols, float* out) {
  __shared__ float sh[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
  if (c < cols) {
    int64_t r = w;
    for (; r + 48 < n; r += 64) {
      const float* p = part + r * stride + c;
      s0 += p[0];
      s1 += p[16 * stride];
      s2 += p[32 * stride];
      s3 += p[48 * stride];
    }
    for (; r < n; r += 16) s0 += part[r * stride + c];
  }
  sh[w][lane] = (s0 + s1) + (s2 + s3);
  __syncthreads();
  if (w == 0 && c < cols) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) s += sh[i][lane];
    out[c] = s;
  }
}

// ---- host: the variant by the row's length.  The fewest lanes that hold a row with a pack each, from 8 on, then more
// packs a lane.  (bf16, 200000 rows of 64 by whole waves, 8 of 64 lanes at work: 61 us.)
struct RowPlan { int tpr, nv; };
// workgroups of a launch: a launch holds fewer than 2^32 threads
unsigned row_blocks(int64_t rows, int tpr) {
  const int64_t n = ceil_div(rows, NT / tpr);
  return (unsigned)(n < (1 << 22) ? n : (1 << 22));
}
RowPlan plan_rows(int dim, int V) {
  for (int tpr = 8; tpr <= 64; tpr *= 2)
    if (dim <= tpr * V) return {tpr, 1};
  for (int nv = 2; nv <= 4; nv *= 2)
    if (dim <= 64 * V * nv) return {64, nv};
  for (int nv = 2; nv <= 8; nv *= 2)
    if (dim <= NT * V * nv) return {NT, nv};
  return {NT, 0};
}
// elements a pack: 16 bytes of T, or one where a row has fewer
int row_pack(int dim, int type) {
  const int W = 16 / type_bytes(type);
  return dim < W ? 1 : W;
}

template <int N> using Int = std::integral_constant<int, N>;
// ALL false: rows of a few elements, one a lane
template <bool ALL, typename F> int32_t by_plan(RowPlan p, F f) {
  if constexpr (ALL) {
    if (p.tpr == 16) return f(Int<16>(), Int<1>());
    if (p.tpr == 32) return f(Int<32>(), Int<1>());
    if (p.tpr == 64) {
      if (p.nv == 1) return f(Int<64>(), Int<1>());
      if (p.nv == 2) return f(Int<64>(), Int<2>());
      return f(Int<64>(), Int<4>());
    }
    if (p.tpr == NT) {
      if (p.nv == 2) return f(Int<NT>(), Int<2>());
      if (p.nv == 4) return f(Int<NT>(), Int<4>());
      if (p.nv == 8) return f(Int<NT>(), Int<8>());
      return f(Int<NT>(), Int<0>());
    }
  }
  return f(Int<8>(), Int<1>());
}

// rows start on a pack's boundary
bool packs(const void* p, int64_t stride, int bytes, int V) {
  return !p || (aligned_to(p, (size_t)bytes * V) && stride % V == 0);
}

template <typename T, typename R, int V, bool EVEN> int32_t launch_fwd(const NormArgs& a, hipStream_t st) {
  const RowPlan p = plan_rows(a.dim, V);
  const unsigned grid = row_blocks(a.rows, p.tpr);
  return by_plan<(V > 1)>(p, [&](auto tpr, auto nv) -> int32_t {
    if (a.q) hipLaunchKernelGGL((norm_fwd_kernel<T, R, V, EVEN, tpr, nv, true>), dim3(grid), dim3(NT), 0, st, a);
    else hipLaunchKernelGGL((norm_fwd_kernel<T, R, V, EVEN, tpr, nv, false>), dim3(grid), dim3(NT), 0, st, a);
    return pnp_check_launch("norm_fwd_kernel");
  });
}

template <typename T, typename R> int32_t run_fwd(const NormArgs& a, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (a.dim < V) return launch_fwd<T, R, 1, true>(a, st);
  const bool even = a.dim % V == 0 && packs(a.x, a.xs, sizeof(T), V) && packs(a.r, a.rs, sizeof(R), V) &&
                    packs(a.w, 0, 4, V) && packs(a.y, a.dim, sizeof(T), V) && packs(a.s, a.dim, sizeof(R), V) &&
                    packs(a.q, a.qs, 1, V);
  return even ? launch_fwd<T, R, V, true>(a, st) : launch_fwd<T, R, V, false>(a, st);
}

// workgroups of the gradient: one a CU, and more as long as their rows of `part` stay small next to what they read
// (8 rows a thread, or more)
int64_t bwd_blocks(int64_t rows, int tpr) {
  const int64_t per = NT / tpr;
  const int64_t want = ceil_div(rows, per * 8), least = ceil_div(rows, per) < 256 ? ceil_div(rows, per) : 256;
  return want < least ? least : want > 1024 ? 1024 : want;
}
constexpr int64_t DW_STRIPS = 64;   // row strips of norm_dw_kernel
int64_t bwd_parts(int64_t rows, int dim, int V) {
  const RowPlan p = plan_rows(dim, V);
  return p.nv ? bwd_blocks(rows, p.tpr) : DW_STRIPS;
}

template <typename T, typename R, int V, bool EVEN> int32_t launch_bwd(NormBwdArgs a, float* dw, hipStream_t st) {
  const RowPlan p = plan_rows(a.dim, V);
  const int64_t grid = bwd_blocks(a.rows, p.tpr);
  int32_t rc = by_plan<(V > 1)>(p, [&](auto tpr, auto nv) -> int32_t {
    hipLaunchKernelGGL((norm_bwd_kernel<T, R, V, EVEN, tpr, nv>), dim3((unsigned)grid), dim3(NT), 0, st, a);
    return pnp_check_launch("norm_bwd_kernel");
  });
  if (rc || !dw) return rc;
  if (!p.nv) {
    hipLaunchKernelGGL((norm_dw_kernel<T, R>), dim3((unsigned)ceil_div(a.dim, NT), DW_STRIPS), dim3(NT), 0, st, a);
    if ((rc = pnp_check_launch("norm_dw_kernel"))) return rc;
  }
  return column_sums(a.part, p.nv ? grid : DW_STRIPS, a.dim, a.dim, dw, st);
}

template <typename T, typename R> int32_t run_bwd(const NormBwdArgs& a, float* dw, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (a.dim < V) return launch_bwd<T, R, 1, true>(a, dw, st);
  const bool even = a.dim % V == 0 && packs(a.dy, a.dys, sizeof(T), V) && packs(a.s, a.ss, sizeof(R), V) &&
                    packs(a.ds, a.dss, sizeof(R), V) && packs(a.w, 0, 4, V) && packs(a.dx, a.dim, sizeof(T), V) &&
                    packs(a.dres, a.dim, sizeof(R), V);
  return even ? launch_bwd<T, R, V, true>(a, dw, st) : launch_bwd<T, R, V, false>(a, dw, st);
}

template <typename T> int32_t run_quantize(const NormArgs& a, hipStream_t st) {
  constexpr int W = 16 / sizeof(T);
  auto go = [&](auto v, auto even) -> int32_t {
    constexpr int V = decltype(v)::value;
    constexpr bool EVEN = decltype(even)::value;
    const RowPlan p = plan_rows(a.dim, V);
    const unsigned grid = row_blocks(a.rows, p.tpr);
    return by_plan<(V > 1)>(p, [&](auto tpr, auto nv) -> int32_t {
      hipLaunchKernelGGL((quantize_kernel<T, V, EVEN, tpr, nv>), dim3(grid), dim3(NT), 0, st, a);
      return pnp_check_launch("quantize_kernel");
    });
  };
  if (a.dim < W) return go(Int<1>(), std::true_type());
  const bool even = a.dim % W == 0 && packs(a.x, a.xs, sizeof(T), W) && packs(a.q, a.qs, 1, W);
  return even ? go(Int<W>(), std::true_type()) : go(Int<W>(), std::false_type());
}

bool rows_ok(int64_t rows, int dim) { return rows >= 0 && rows <= ((int64_t)1 << 40) && dim > 0 && dim <= (1 << 24); }

}  // namespace

int32_t column_sums(const float* part, int64_t n, int64_t stride, int64_t cols, float* out, hipStream_t st) {
  hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)ceil_div(cols, 64)), dim3(1024), 0, st, part, n, stride, cols, out);
  return pnp_check_launch("column_sums_kernel");
}

}  // namespace seq

using namespace seq;

extern "C" int32_t pnp_rms_norm(const pnp_norm_desc* d, void* stream) {
  const char* fn = "pnp_rms_norm";
  if (!d || !rows_ok(d->rows, d->dim) || !type_bytes(d->type) || (d->res_type != d->type && d->res_type != PNP_F32)) {
    pnp_set_error("%s: bad shape or type", fn);
    return PNP_ERR_ARG;
  }
  if (!d->rows) return PNP_OK;
  if (!d->x || (!d->y) == (!d->q) || (d->q && (!d->scale || d->q_stride < d->dim)) || (d->residual && !d->s)) {
    pnp_set_error("%s: null buffer, or not one of y and q", fn);
    return PNP_ERR_ARG;
  }
  if (!d->residual && d->s && d->res_type != d->type) {
    pnp_set_error("%s: the stream alone is in its own type", fn);
    return PNP_ERR_ARG;
  }
  NormArgs a{d->rows, d->x_stride, d->r_stride, d->q_stride, d->dim, d->eps, d->x, d->residual, d->weight, d->y, d->s,
             d->rstd, d->q, d->scale};
  const hipStream_t st = (hipStream_t)stream;
  if (d->res_type == d->type) return SEQ_BY_TYPE(d->type, T, return (run_fwd<T, T>(a, st)));
  return SEQ_BY_TYPE(d->type, T, return (run_fwd<T, float>(a, st)));
}

extern "C" int64_t pnp_rms_norm_bwd_workspace(const pnp_norm_bwd_desc* d) {
  if (!d || !rows_ok(d->rows, d->dim) || !type_bytes(d->type)) {
    pnp_set_error("pnp_rms_norm_bwd_workspace: bad shape or type");
    return PNP_ERR_ARG;
  }
  if (!d->rows) return 0;
  return bwd_parts(d->rows, d->dim, row_pack(d->dim, d->type)) * d->dim;
}

extern "C" int32_t pnp_rms_norm_bwd(const pnp_norm_bwd_desc* d, void* stream) {
  const char* fn = "pnp_rms_norm_bwd";
  if (!d || !rows_ok(d->rows, d->dim) || !type_bytes(d->type) || (d->res_type != d->type && d->res_type != PNP_F32)) {
    pnp_set_error("%s: bad shape or type", fn);
    return PNP_ERR_ARG;
  }
  const hipStream_t st = (hipStream_t)stream;
  if (!d->rows) return d->dweight ? column_sums(nullptr, 0, 0, d->dim, d->dweight, st) : PNP_OK;
  if (!d->dy || !d->s || !d->rstd || !d->dx) {
    pnp_set_error("%s: null buffer", fn);
    return PNP_ERR_ARG;
  }
  if (d->dweight && (!d->workspace || d->workspace_floats < pnp_rms_norm_bwd_workspace(d))) {
    pnp_set_error("%s: workspace too small", fn);
    return PNP_ERR_ARG;
  }
  NormBwdArgs a{d->rows, d->dy_stride, d->ds_stride, d->s_stride, d->dim, d->dy, d->ds, d->s, d->weight, d->rstd,
                d->dx, d->dres, d->dweight ? d->workspace : nullptr};
  if (d->res_type == d->type) return SEQ_BY_TYPE(d->type, T, return (run_bwd<T, T>(a, d->dweight, st)));
  return SEQ_BY_TYPE(d->type, T, return (run_bwd<T, float>(a, d->dweight, st)));
}

extern "C" int32_t pnp_quantize_rows(const void* x, int64_t x_stride, int32_t type, int64_t rows, int32_t dim, int8_t* q,
                                     int64_t q_stride, float* scale, void* stream) {
  if (!rows_ok(rows, dim) || !type_bytes(type) || q_stride < dim) {
    pnp_set_error("pnp_quantize_rows: bad shape or type");
    return PNP_ERR_ARG;
  }
  if (!rows) return PNP_OK;
  if (!x || !q || !scale) {
    pnp_set_error("pnp_quantize_rows: null buffer");
    return PNP_ERR_ARG;
  }
  NormArgs a{};
  a.rows = rows; a.xs = x_stride; a.qs = q_stride; a.dim = dim; a.x = x; a.q = q; a.scale = scale;
  const hipStream_t st = (hipStream_t)stream;
  return SEQ_BY_TYPE(type, T, return run_quantize<T>(a, st));
}
