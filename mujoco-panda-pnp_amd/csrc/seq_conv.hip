// seq_conv.hip — the short causal convolution along a sequence, one filter per channel: forward,
// gradient, and the single-token form (include/pnp.h pnp_causal_conv and its kin).
//
//   pre[t] = bias + sum_{j < W} w[j] x[t - W + 1 + j],  y = pre or pre sigmoid(pre)
//   dx[t] = sum_{k < W} w[W - 1 - k] dpre[t + k],  dw[j] = sum dpre[t] x[t - W + 1 + j],  dbias = sum dpre
//
// where a tap reaches past the start of its sequence it is dropped.  Bound by HBM: a lane holds V
// neighbouring channels and walks a run of tokens with the last W - 1 of them in registers, so a token
// is read once but for the runs' ends.
#include <type_traits>

#include "seq_dev.h"

namespace seq {
namespace {

constexpr int NT = 256;

struct ConvArgs {
  int64_t B, L, xb, xt;
  int dim, silu;
  int64_t runs;      // runs of a sequence
  int run;           // tokens of a run
  const void* x;
  const float *w, *bias;
  const uint8_t* starts;
  const void* state;
  void *y, *last;
};

template <int V, typename T> __device__ __forceinline__ void read_token(const ConvArgs& a, const T* x, const T* state, int W, int64_t b,
                                                                        int64_t t, int c, float (&v)[V]) {
  if (t >= 0) load_f<V>(x + b * a.xb + t * a.xt + c, v);
  else if (state && t >= -(W - 1)) load_f<V>(state + (b * (W - 1) + t + W - 1) * a.dim + c, v);
  else
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = 0.f;
}

// h: the last W - 1 tokens, oldest first
template <int W, int V> __device__ __forceinline__ void push(float (&h)[W - 1][V], const float (&v)[V]) {
#pragma unroll
  for (int j = 0; j + 1 < W - 1; j++)
#pragma unroll
    for (int i = 0; i < V; i++) h[j][i] = h[j + 1][i];
#pragma unroll
  for (int i = 0; i < V; i++) h[W - 2][i] = v[i];
}
template <int W, int V> __device__ __forceinline__ void clear(float (&h)[W - 1][V]) {
#pragma unroll
  for (int j = 0; j < W - 1; j++)
#pragma unroll
    for (int i = 0; i < V; i++) h[j][i] = 0.f;
}
// the W - 1 tokens before t0, those before a start at or before t0 - 1 as zeros
template <int W, int V, typename T> __device__ __forceinline__ void history(const ConvArgs& a, const T* x, const T* state, int64_t b,
                                                                            int64_t t0, int c, float (&h)[W - 1][V]) {
  clear<W, V>(h);
#pragma unroll
  for (int j = 0; j < W - 1; j++) {
    const int64_t t = t0 - (W - 1) + j;
    float v[V];
    read_token<V>(a, x, state, W, b, t, c, v);
    if (a.starts && t >= 0 && a.starts[b * a.L + t]) clear<W, V>(h);
    push<W, V>(h, v);
  }
}

template <int W, int V> __device__ __forceinline__ void taps(const float* w, const float* bias, int c, float (&wt)[W][V], float (&bs)[V]) {
#pragma unroll
  for (int i = 0; i < V; i++) {
#pragma unroll
    for (int j = 0; j < W; j++) wt[j][i] = w[(int64_t)(c + i) * W + j];
    bs[i] = bias ? bias[c + i] : 0.f;
  }
}

// pre of a token whose W - 1 predecessors are h
template <int W, int V>
__device__ __forceinline__ void tap_sum(const float (&wt)[W][V], const float (&bs)[V], const float (&h)[W - 1][V], const float (&v)[V],
                                        float (&pre)[V]) {
#pragma unroll
  for (int i = 0; i < V; i++) {
    float p = bs[i];
#pragma unroll
    for (int j = 0; j < W - 1; j++) p += wt[j][i] * h[j][i];
    pre[i] = p + wt[W - 1][i] * v[i];
  }
}

// A lane: V channels of one run.  Lanes of a wave lie along the channels first.  The next TB tokens are
// loaded before the first of these is used: the stores between would hold their loads back.
// Bf16, 2 x 8191 x 2048: 30 us, 134 MB at 4.4 TB/s (a large copy's 5.1); eight tokens ahead gain nothing.
constexpr int TB = 4;
template <typename T, int W, int V> __global__ __launch_bounds__(NT) void conv_fwd_kernel(ConvArgs a) {
  const int64_t packs = a.dim / V, id = (int64_t)blockIdx.x * NT + threadIdx.x;
  const int64_t k = id / packs;
  if (k >= a.B * a.runs) return;
  const int c = (int)(id - k * packs) * V;
  const int64_t b = k / a.runs, t0 = (k - b * a.runs) * a.run, t1 = t0 + a.run < a.L ? t0 + a.run : a.L;
  const T *x = (const T*)a.x, *state = (const T*)a.state;
  float wt[W][V], bs[V], h[W - 1][V];
  taps<W, V>(a.w, a.bias, c, wt, bs);
  history<W, V>(a, x, state, b, t0, c, h);
  const T* px = x + b * a.xb + t0 * a.xt + c;
  T* py = (T*)a.y + (b * a.L + t0) * a.dim + c;
  const uint8_t* ps = a.starts ? a.starts + b * a.L : nullptr;
  Pack<T, V> next[TB], raw[TB];
  bool ns[TB], st[TB];
  auto fetch = [&](int64_t t) {
#pragma unroll
    for (int k = 0; k < TB; k++)
      if (t + k < t1) {
        next[k] = *reinterpret_cast<const Pack<T, V>*>(px + k * a.xt);
        ns[k] = ps && ps[t + k];
      }
    px += TB * a.xt;
  };
  fetch(t0);
  for (int64_t t = t0; t < t1; t += TB, py += (int64_t)TB * a.dim) {
#pragma unroll
    for (int k = 0; k < TB; k++) {
      raw[k] = next[k];
      st[k] = ns[k];
    }
    fetch(t + TB);
#pragma unroll
    for (int k = 0; k < TB; k++) {
      if (t + k >= t1) break;
      float v[V], pre[V];
#pragma unroll
      for (int i = 0; i < V; i++) v[i] = to_f(raw[k].v[i]);
      if (st[k]) clear<W, V>(h);
      tap_sum<W, V>(wt, bs, h, v, pre);
      if (a.silu)
#pragma unroll
        for (int i = 0; i < V; i++) pre[i] *= sigmoid_f(pre[i]);
      store_f<V>(py + (int64_t)k * a.dim, pre);
      push<W, V>(h, v);
    }
  }
  if (a.last && t1 == a.L)
#pragma unroll
    for (int j = 0; j < W - 1; j++) store_f<V>((T*)a.last + (b * (W - 1) + j) * a.dim + c, h[j]);
}

struct ConvBwdArgs {
  ConvArgs f;
  int64_t dyb, dyt, parts;   // parts: workgroup rows of the weights' sums
  const void *dy, *dlast;
  void *dx, *dstate;
  float* part;               // [parts][dim][W + 1]
};

// A workgroup: 4 waves on the same 64 packs of channels, a run of tokens each, and on to the run
// `parts * 4` further; the weights' gradients stay in registers over all of a wave's runs and leave,
// summed over the 4 waves in their order, as one row of `part`.
//
// A token's dx needs the dpre of the W - 1 tokens after it: the walk goes W - 1 tokens past the run's
// end, and dx is written W - 1 tokens behind.  acc[k] holds the sum for token t - k; tokens before the
// start of t's sequence get nothing from it (age: tokens since the start).
//
// Four channels a lane: with eight the filters and sums spill (bf16, 2 x 8191 x 2048: 125 against 59 us).  The tokens
// within a run and its sequence go without the questions that the run's ends ask (59 -> 49 us, 201 MB at 4.1 TB/s).
// Channels that are no multiple of 4, one a lane, with the weights' sums: bf16, 2 x 4096 x 2047, 40 us, x 2048 29 and x 2044
// (by fours, rows across lines) 37.
template <typename T, int W, int V> __global__ __launch_bounds__(NT, 2) void conv_bwd_kernel(ConvBwdArgs a) {
  const ConvArgs& f = a.f;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // (a wave's run, its marks and its age are scalars)
  const int npack = f.dim / V;
  const int pk = blockIdx.x * 64 + lane;
  const bool on = pk < npack;
  const int c = (on ? pk : npack - 1) * V;
  const uint32_t cb = (uint32_t)c * sizeof(T);
  const T *x = (const T*)f.x, *state = (const T*)f.state, *dy = (const T*)a.dy, *dlast = (const T*)a.dlast;
  float wt[W][V], bs[V], dw[W][V] = {}, db[V] = {};
  taps<W, V>(f.w, f.bias, c, wt, bs);
  for (int64_t k = (int64_t)blockIdx.y * 4 + wave; k < f.B * f.runs; k += (int64_t)gridDim.y * 4) {
    const int64_t b = k / f.runs, t0 = (k - b * f.runs) * f.run, t1 = t0 + f.run < f.L ? t0 + f.run : f.L;
    const uint8_t* ps = f.starts ? f.starts + b * f.L : nullptr;
    float h[W - 1][V], acc[W][V];
    history<W, V>(f, x, state, b, t0, c, h);
#pragma unroll
    for (int j = 0; j < W; j++)
#pragma unroll
      for (int i = 0; i < V; i++) acc[j][i] = 0.f;
    // the run that begins the sequence writes the gradient of the state too
    const int64_t first = t0 == 0 ? -(W - 1) : t0;
    int age = W - 1;
    if (ps)   // the distance to the last start among the W - 1 tokens before t0
#pragma unroll
      for (int j = W - 1; j >= 1; j--)
        if (t0 - j >= 0 && ps[t0 - j]) age = j - 1;
    const T *px = x + b * f.xb + t0 * f.xt, *pg = dy + b * a.dyb + t0 * a.dyt;   // (scalars; the lane's channels are at + cb)
    T* po = (T*)a.dx + (b * f.L + t0 - (W - 1)) * f.dim;
    const int64_t end = t1 + W - 1, held = end < f.L ? end : f.L;   // the walk's end, and the last token there is for it
    Pack<T, V> nx[TB], ng[TB], rx[TB], rg[TB];
    bool nm[TB], mark[TB];
    auto fetch = [&](int64_t tb) {
#pragma unroll
      for (int k = 0; k < TB; k++) {
        if (tb + k < held) {
          nx[k] = *reinterpret_cast<const Pack<T, V>*>(at<T>(px, 0, cb));
          ng[k] = *reinterpret_cast<const Pack<T, V>*>(at<T>(pg, 0, cb));
          nm[k] = ps && ps[tb + k];
        }
        px += f.xt;
        pg += a.dyt;
      }
    };
    // ALL: a token of the run, its predecessors of its sequence all (age W - 1), and its oldest predecessor the run's too
    auto token = [&](auto all, int64_t t, const Pack<T, V>& xk, const Pack<T, V>& gk, bool start) {
      constexpr bool ALL = decltype(all)::value;
      if (ALL || t < f.L) {
        float v[V], g[V], pre[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
          v[i] = to_f(xk.v[i]);
          g[i] = to_f(gk.v[i]);
        }
        if (!ALL && start) {
          clear<W, V>(h);
          age = 0;
        } else if (!ALL && age < W - 1) {
          age++;
        }
        if (f.silu) {
          tap_sum<W, V>(wt, bs, h, v, pre);
#pragma unroll
          for (int i = 0; i < V; i++) {
            const float s = sigmoid_f(pre[i]);
            g[i] *= s * (1.f + pre[i] * (1.f - s));
          }
        }
        if (ALL || t < t1) {
#pragma unroll
          for (int i = 0; i < V; i++) {
#pragma unroll
            for (int j = 0; j < W - 1; j++) dw[j][i] += g[i] * h[j][i];
            dw[W - 1][i] += g[i] * v[i];
            db[i] += g[i];
          }
        }
#pragma unroll
        for (int j = 0; j < W; j++)
          if (ALL || j <= age)
#pragma unroll
            for (int i = 0; i < V; i++) acc[j][i] += wt[W - 1 - j][i] * g[i];
        push<W, V>(h, v);
      } else if (age < W - 1) {
        age++;
      }
      // what last_state's gradient brings, at the walk's first token past the last: its row W - 1 - j is token L - j,
      // held in acc[j], if that still belongs to the sequence
      if (!ALL && dlast && t == f.L) {
#pragma unroll
        for (int j = 1; j < W; j++)
          if (j <= age) {
            float g[V];
            load_f<V>(dlast + (b * (W - 1) + W - 1 - j) * f.dim + c, g);
#pragma unroll
            for (int i = 0; i < V; i++) acc[j][i] += g[i];
          }
      }
      const int64_t o = t - (W - 1);
      if (on && (ALL || (o >= first && o < t1))) {
        if (ALL || o >= 0) store_f<V>(at<T>(po, 0, cb), acc[W - 1]);
        else if (a.dstate) store_f<V>((T*)a.dstate + (b * (W - 1) + o + W - 1) * f.dim + c, acc[W - 1]);
      }
      po += f.dim;
#pragma unroll
      for (int j = W - 1; j > 0; j--)
#pragma unroll
        for (int i = 0; i < V; i++) acc[j][i] = acc[j - 1][i];
#pragma unroll
      for (int i = 0; i < V; i++) acc[0][i] = 0.f;
    };
    fetch(t0);
    for (int64_t tb = t0; tb < end; tb += TB) {
      bool marked = false;
#pragma unroll
      for (int k = 0; k < TB; k++) {
        rx[k] = nx[k];
        rg[k] = ng[k];
        mark[k] = nm[k];
        marked |= tb + k < held && mark[k];
      }
      fetch(tb + TB);
      if (tb - t0 >= W - 1 && tb + TB <= t1 && age == W - 1 && !marked) {
#pragma unroll
        for (int k = 0; k < TB; k++) token(std::true_type(), tb + k, rx[k], rg[k], false);
      } else {
#pragma unroll
        for (int k = 0; k < TB; k++)
          if (tb + k < end) token(std::false_type(), tb + k, rx[k], rg[k], mark[k]);
      }
    }
  }
  if (!a.part) return;
  __shared__ float sh[3][64][V];
#pragma unroll
  for (int j = 0; j <= W; j++) {
    float s[V];
#pragma unroll
    for (int i = 0; i < V; i++) s[i] = j < W ? dw[j < W ? j : 0][i] : db[i];
    if (wave)
#pragma unroll
      for (int i = 0; i < V; i++) sh[wave - 1][lane][i] = s[i];
    __syncthreads();
    if (!wave && on) {
#pragma unroll
      for (int i = 0; i < V; i++)
        a.part[((int64_t)blockIdx.y * (W + 1) + j) * f.dim + c + i] = s[i] + sh[0][lane][i] + sh[1][lane][i] + sh[2][lane][i];
    }
    __syncthreads();
  }
}

// dweight [dim][W] and dbias [dim] from part [parts][W + 1][dim]
__global__ __launch_bounds__(1024) void conv_dw_kernel(const float* part, int64_t parts, int dim, int W, float* dw, float* db) {
  __shared__ float sh[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, j = blockIdx.y;
  const int c = blockIdx.x * 64 + lane;
  float s0 = 0.f, s1 = 0.f;
  if (c < dim) {
    int64_t r = w;
    for (; r + 16 < parts; r += 32) {
      s0 += part[(r * (W + 1) + j) * dim + c];
      s1 += part[((r + 16) * (W + 1) + j) * dim + c];
    }
    if (r < parts) s0 += part[(r * (W + 1) + j) * dim + c];
  }
  sh[w][lane] = s0 + s1;
  __syncthreads();
  if (w || c >= dim) return;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i++) s += sh[i][lane];
  if (j == W) { if (db) db[c] = s; }
  else if (dw) dw[(int64_t)c * W + j] = s;
}

struct ConvStepArgs {
  int64_t B, xs;
  int dim, silu;
  const void* x;
  void* state;
  const float *w, *bias;
  const uint8_t* reset;
  void* y;
};
// One token: the state moves up by one in place.  Bound by memory: fp32, 8192 x 512, W 4, 21 us, 134 MB at 6.3 TB/s.
template <typename T, int W, int V> __global__ __launch_bounds__(NT) void conv_step_kernel(ConvStepArgs a) {
  const int64_t packs = a.dim / V;
  for (int64_t id = (int64_t)blockIdx.x * NT + threadIdx.x; id < a.B * packs; id += (int64_t)gridDim.x * NT) {
    const int64_t b = id / packs;
    const int c = (int)(id - b * packs) * V;
    T* st = (T*)a.state + b * (W - 1) * a.dim + c;
    float wt[W][V], bs[V], h[W - 1][V], v[V], pre[V];
    load_f<V>((const T*)a.x + b * a.xs + c, v);
#pragma unroll
    for (int j = 0; j < W - 1; j++) load_f<V>(st + (int64_t)j * a.dim, h[j]);
    taps<W, V>(a.w, a.bias, c, wt, bs);
    if (a.reset && a.reset[b]) clear<W, V>(h);
    tap_sum<W, V>(wt, bs, h, v, pre);
    if (a.silu)
#pragma unroll
      for (int i = 0; i < V; i++) pre[i] *= sigmoid_f(pre[i]);
    store_f<V>((T*)a.y + b * a.dim + c, pre);
    push<W, V>(h, v);
#pragma unroll
    for (int j = 0; j < W - 1; j++) store_f<V>(st + (int64_t)j * a.dim, h[j]);
  }
}

// ---- host
template <typename F> int32_t by_width(int W, F f) {
  if (W == 2) return f(std::integral_constant<int, 2>());
  if (W == 3) return f(std::integral_constant<int, 3>());
  return f(std::integral_constant<int, 4>());
}
bool on_pack(const void* p, size_t bytes) { return !p || aligned_to(p, bytes); }

constexpr int VB = 4;         // channels a lane of the gradient: the filters, their sums and the tokens under them in registers
// tokens of a run: long enough that the W - 1 tokens a run reads twice are few, short enough for 2 waves a SIMD,
// a sequence's runs of one length
int run_length(int64_t B, int64_t L, int64_t packs) {
  int run = 64;
  while (run > 8 && B * ceil_div(L, run) * packs < 128 * 1024) run /= 2;
  return L ? (int)ceil_div(L, ceil_div(L, run)) : run;
}
int64_t bwd_parts(int64_t B, int64_t L, int64_t packs, int run) {
  const int64_t cols = ceil_div(packs, 64), rows = ceil_div(B * ceil_div(L, run), 4);
  const int64_t most = ceil_div(2048, cols);
  return rows < 1 ? 1 : rows < most ? rows : most;
}

bool conv_ok(const pnp_conv_desc* d) {
  return d && d->B >= 0 && d->L >= 0 && d->dim > 0 && d->dim <= (1 << 24) && d->width >= 2 && d->width <= 4 &&
         type_bytes(d->type) && d->B <= ((int64_t)1 << 31) && d->L <= ((int64_t)1 << 31);
}
ConvArgs conv_args(const pnp_conv_desc* d) {
  ConvArgs a{};
  a.B = d->B; a.L = d->L; a.xb = d->x_bstride; a.xt = d->x_tstride; a.dim = d->dim; a.silu = d->silu;
  a.x = d->x; a.w = d->weight; a.bias = d->bias; a.starts = d->starts; a.state = d->state; a.y = d->y; a.last = d->last_state;
  return a;
}

template <typename T, int V> int32_t launch_conv(ConvArgs a, int W, hipStream_t st) {
  const int64_t packs = a.dim / V;
  a.run = run_length(a.B, a.L, packs);
  a.runs = a.L ? ceil_div(a.L, a.run) : 1;   // a sequence of no tokens still hands its state on
  const int64_t grid = ceil_div(a.B * a.runs * packs, NT);
  if (grid >= (1 << 24)) { pnp_set_error("pnp_causal_conv: too many tokens for one launch"); return PNP_ERR_ARG; }
  return by_width(W, [&](auto w) -> int32_t {
    hipLaunchKernelGGL((conv_fwd_kernel<T, w, V>), dim3((unsigned)grid), dim3(NT), 0, st, a);
    return pnp_check_launch("conv_fwd_kernel");
  });
}
template <typename T> int32_t run_conv(const ConvArgs& a, int W, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = a.dim % V == 0 && a.xb % V == 0 && a.xt % V == 0 && on_pack(a.x, 16) && on_pack(a.state, 16) &&
                    on_pack(a.y, 16) && on_pack(a.last, 16);
  return wide ? launch_conv<T, V>(a, W, st) : launch_conv<T, 1>(a, W, st);
}

template <typename T, int V> int32_t launch_conv_bwd(ConvBwdArgs a, int W, float* dw, float* db, hipStream_t st) {
  const int64_t packs = a.f.dim / V;
  a.f.run = run_length(a.f.B, a.f.L, packs);
  a.f.runs = a.f.L ? ceil_div(a.f.L, a.f.run) : 1;
  a.parts = bwd_parts(a.f.B, a.f.L, packs, a.f.run);
  const int32_t rc = by_width(W, [&](auto w) -> int32_t {
    hipLaunchKernelGGL((conv_bwd_kernel<T, w, V>), dim3((unsigned)ceil_div(packs, 64), (unsigned)a.parts), dim3(NT), 0, st, a);
    return pnp_check_launch("conv_bwd_kernel");
  });
  if (rc || !a.part) return rc;
  hipLaunchKernelGGL(conv_dw_kernel, dim3((unsigned)ceil_div(a.f.dim, 64), (unsigned)(W + 1)), dim3(1024), 0, st, a.part, a.parts, a.f.dim,
                     W, dw, db);
  return pnp_check_launch("conv_dw_kernel");
}
template <typename T> int32_t run_conv_bwd(const ConvBwdArgs& a, int W, float* dw, float* db, hipStream_t st) {
  constexpr size_t by = VB * sizeof(T);
  const bool wide = a.f.dim % VB == 0 && a.f.xb % VB == 0 && a.f.xt % VB == 0 && a.dyb % VB == 0 && a.dyt % VB == 0 &&
                    on_pack(a.f.x, by) && on_pack(a.f.state, by) && on_pack(a.dy, by) && on_pack(a.dlast, by) &&
                    on_pack(a.dx, by) && on_pack(a.dstate, by);
  return wide ? launch_conv_bwd<T, VB>(a, W, dw, db, st) : launch_conv_bwd<T, 1>(a, W, dw, db, st);
}

template <typename T> int32_t run_conv_step(const ConvStepArgs& a, int W, hipStream_t st) {
  constexpr int WIDE = 16 / sizeof(T);
  auto go = [&](auto v) -> int32_t {
    constexpr int V = decltype(v)::value;
    const int64_t n = ceil_div(a.B * (a.dim / V), NT);
    const unsigned grid = (unsigned)(n < (1 << 22) ? n : (1 << 22));
    return by_width(W, [&](auto w) -> int32_t {
      hipLaunchKernelGGL((conv_step_kernel<T, w, V>), dim3(grid), dim3(NT), 0, st, a);
      return pnp_check_launch("conv_step_kernel");
    });
  };
  const bool wide = a.dim % WIDE == 0 && a.xs % WIDE == 0 && on_pack(a.x, 16) && on_pack(a.state, 16) && on_pack(a.y, 16);
  return wide ? go(std::integral_constant<int, WIDE>()) : go(std::integral_constant<int, 1>());
}

}  // namespace
}  // namespace seq

using namespace seq;

extern "C" int32_t pnp_causal_conv(const pnp_conv_desc* d, void* stream) {
  const char* fn = "pnp_causal_conv";
  if (!conv_ok(d)) {
    pnp_set_error("%s: bad shape, width or type", fn);
    return PNP_ERR_ARG;
  }
  if (!d->B || (!d->L && !d->last_state)) return PNP_OK;
  if (!d->weight || (d->L && (!d->x || !d->y))) {
    pnp_set_error("%s: null buffer", fn);
    return PNP_ERR_ARG;
  }
  const ConvArgs a = conv_args(d);
  const hipStream_t st = (hipStream_t)stream;
  return SEQ_BY_TYPE(d->type, T, return run_conv<T>(a, d->width, st));
}

extern "C" int64_t pnp_causal_conv_bwd_workspace(const pnp_conv_bwd_desc* d) {
  if (!d || !conv_ok(&d->f)) {
    pnp_set_error("pnp_causal_conv_bwd_workspace: bad shape, width or type");
    return PNP_ERR_ARG;
  }
  const pnp_conv_desc& f = d->f;
  if (!f.B) return 0;
  int64_t most = 0;   // whichever of the two loads the tensors' alignment leads to
  for (int V : {VB, 1}) {
    const int64_t packs = ceil_div(f.dim, V);
    const int64_t n = bwd_parts(f.B, f.L ? f.L : 1, packs, run_length(f.B, f.L, packs));
    if (n > most) most = n;
  }
  return most * f.dim * (f.width + 1);
}

extern "C" int32_t pnp_causal_conv_bwd(const pnp_conv_bwd_desc* d, void* stream) {
  const char* fn = "pnp_causal_conv_bwd";
  if (!d || !conv_ok(&d->f)) {
    pnp_set_error("%s: bad shape, width or type", fn);
    return PNP_ERR_ARG;
  }
  const pnp_conv_desc& f = d->f;
  const hipStream_t st = (hipStream_t)stream;
  if (!f.B) {
    if (!d->dweight && !d->dbias) return PNP_OK;
    hipLaunchKernelGGL(conv_dw_kernel, dim3((unsigned)ceil_div(f.dim, 64), (unsigned)(f.width + 1)), dim3(1024), 0, st,
                       (const float*)nullptr, (int64_t)0, f.dim, f.width, d->dweight, d->dbias);
    return pnp_check_launch("conv_dw_kernel");
  }
  if (!f.weight || (f.L && (!f.x || !d->dy || !d->dx))) {
    pnp_set_error("%s: null buffer", fn);
    return PNP_ERR_ARG;
  }
  const bool sums = d->dweight || d->dbias;
  if (sums && (!d->workspace || d->workspace_floats < pnp_causal_conv_bwd_workspace(d))) {
    pnp_set_error("%s: workspace too small", fn);
    return PNP_ERR_ARG;
  }
  ConvBwdArgs a{};
  a.f = conv_args(&f);
  a.dyb = d->dy_bstride; a.dyt = d->dy_tstride; a.dy = d->dy; a.dlast = d->dlast; a.dx = d->dx; a.dstate = d->dstate;
  a.part = sums ? d->workspace : nullptr;
  return SEQ_BY_TYPE(f.type, T, return run_conv_bwd<T>(a, f.width, d->dweight, d->dbias, st));
}

extern "C" int32_t pnp_causal_conv_step(const void* x, int64_t x_stride, void* state, const float* weight, const float* bias,
                                        const uint8_t* reset, int64_t B, int32_t dim, int32_t width, int32_t type, int32_t silu,
                                        void* y, void* stream) {
  const char* fn = "pnp_causal_conv_step";
  if (B < 0 || B > ((int64_t)1 << 31) || dim <= 0 || dim > (1 << 24) || width < 2 || width > 4 || !type_bytes(type)) {
    pnp_set_error("%s: bad shape, width or type", fn);
    return PNP_ERR_ARG;
  }
  if (!B) return PNP_OK;
  if (!x || !state || !weight || !y) {
    pnp_set_error("%s: null buffer", fn);
    return PNP_ERR_ARG;
  }
  ConvStepArgs a{B, x_stride, dim, silu, x, state, weight, bias, reset, y};
  const hipStream_t st = (hipStream_t)stream;
  return SEQ_BY_TYPE(type, T, return run_conv_step<T>(a, width, st));
}
