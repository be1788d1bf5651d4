// seq_scan.hip — the selective state space scan: forward, gradient, and the single-token form
// (include/pnp.h pnp_selective_scan and its kin).
//
//   dt = softplus(delta + bias), a = exp(dt A), h[t] = a h[t-1] + dt u B, y = sum_n C h + D u,
//   out = y z sigmoid(z); a = 0 at a token that starts a sequence.
// With dy = dout z sigmoid(z) and g[t] = C dy + a[t+1] g[t+1]:
//   dC = sum_d dy h, dB = sum_d g dt u, du = D dy + dt sum_n g B,
//   ddt = sum_n g (a h[t-1]) A + u sum_n g B, ddelta = ddt sigmoid(delta + bias),
//   dA = sum_{b,t} g dt (a h[t-1]), dD = sum dy u, dz = dout y sigmoid(z) (1 + z (1 - sigmoid(z)))
//
// Layout: a lane holds 4 states of one channel, S = ceil(N / 4) lanes (a power of two) a channel, so a
// wave has 64 / S channels and a workgroup of 4 waves CW = 256 / S.  The workgroup walks its channels
// along the length in tiles: it loads a tile of u, delta, z whole lines at a time, turns them into
// dt and dt u once (a lane's S - 1 neighbours would repeat the softplus), and leaves them in LDS with
// the tile's B and C, which all its channels share.  The next tile's loads are in flight meanwhile.
//
// Per state and token the recurrence costs one exp2 (a quarter-rate instruction: 4) and 4 more
// instructions; with N = 16 that, not HBM, bounds it.
//
// Few sequences of great length do not fill the chip: the length is cut in chunks, a first pass gets
// each chunk's state from a zero start and its decay (exp(A sum dt): one number a channel), a small
// kernel chains them, and the main pass starts every chunk from its true state.  The gradient does the
// same from the other end.
#include <type_traits>

#include "seq_dev.h"

namespace seq {
namespace {

constexpr int NT = 256;

// tokens of a tile, forward and gradient; the gradient's inner tile, whose states and decays stay in
// registers (8 a token), is TR tokens: the forward keeps a state for each
constexpr int tile_f(int S, int bytes) {   // 4 or 8 channels a thread: registers for 4 waves a SIMD
  return S == 1 ? 8 : S == 2 ? (bytes == 4 ? 8 : 16) : S == 4 ? (bytes == 4 ? 16 : 32) : 32;
}
// (N 5 .. 8, fp32: 16 tokens spill, 512 x 33 x 512 x 8 forward and gradient 195 us against 165; bf16, 4 x 2048 x 2048 x 8,
// 305 against 313 the other way.  N 16, fp32 and bf16: 271 and 471 us by 16 tokens, 279 and 502 by 8.)
constexpr int tile_b(int S, int bytes) { return S == 1 || (S == 2 && bytes == 4) ? 8 : 16; }
constexpr int TR = 8;
// waves a SIMD that the forward is built for: what its registers allow without spills
constexpr int fwd_waves(int S, int bytes) { return S >= 8 || (S == 1 && bytes == 4) ? 3 : 4; }

struct ScanArgs {
  int64_t B, L;
  int dim, N, groups, per;       // per: channels of a group
  int tiles;                     // workgroups across a group's channels
  int nch;                       // chunks of the length
  int64_t chunk;                 // tokens of a chunk, a multiple of TR
  int64_t nck;                   // states kept a sequence: one each TR tokens
  const void *u, *delta, *z, *Bm, *Cm;
  int64_t ub, ut, db, dt, zb, zt, Bb, Bt, Cb, Ct;
  const float *A, *D, *bias, *state;
  const uint8_t* starts;
  void* out;
  float *last, *ckpt;
  float *hin;                    // [B][nch][dim][4 S] states at the chunks' starts (nch > 1)
  float *dsum;                   // [B][nch][dim] sums of dt; NaN where the chunk holds a start
};

struct Where { int64_t b, row; int chunk, g, c0, ch; };   // c0: first channel within the group; row: b * nch + chunk
// the workgroup's place among the sequences' chunks [first, first + chunks)
template <int S> __device__ __forceinline__ Where where(const ScanArgs& a, int first, int chunks) {
  const uint32_t per_row = a.groups * a.tiles, row = blockIdx.x / per_row, r = blockIdx.x - row * per_row;
  Where w;
  w.b = row / (uint32_t)chunks;
  w.chunk = (int)(row - (uint32_t)w.b * chunks) + first;
  w.row = w.b * a.nch + w.chunk;
  w.g = (int)r / a.tiles;
  w.c0 = ((int)r - w.g * a.tiles) * (NT / S);
  w.ch = w.g * a.per + w.c0;
  return w;
}

// E neighbouring channels of one token; those past `left` as 0.  WIDE: packs of V are whole or past it, and on their
// boundaries; otherwise whole ones come from wherever they lie, the last channels one by one (by elements throughout,
// bf16, 2 x 2048 x 2047 x 16: 127 us forward, 204 back).
template <typename T, int E> struct Raw { T v[E]; };
template <int E, bool WIDE, typename T> __device__ __forceinline__ void load_channels(const T* p, int left, Raw<T, E>& o) {
  constexpr int V = E * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : E;
#pragma unroll
  for (int i = 0; i < E; i += V) {
    typename PackOf<T, V, WIDE>::type w;
#pragma unroll
    for (int k = 0; k < V; k++) w.v[k] = (T)0.f;
    if constexpr (WIDE) {
      if (i < left) w = *reinterpret_cast<const Pack<T, V>*>(p + i);
    } else if (i + V <= left) {
      w = *reinterpret_cast<const LoosePack<T, V>*>(p + i);
    } else {
#pragma unroll
      for (int k = 0; k < V - 1; k++)
        if (i + k < left) w.v[k] = p[i + k];
    }
#pragma unroll
    for (int k = 0; k < V; k++) o.v[i + k] = w.v[k];
  }
}
template <int E, bool WIDE, typename T> __device__ __forceinline__ void store_channels(T* p, int left, const float (&v)[E]) {
  constexpr int V = E * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : E;
#pragma unroll
  for (int i = 0; i < E; i += V) {
    float w[V];
#pragma unroll
    for (int k = 0; k < V; k++) w[k] = v[i + k];
    if (WIDE ? i < left : i + V <= left) store_f<V, WIDE>(p + i, w);
    else if (!WIDE && i < left)
#pragma unroll
      for (int k = 0; k < V; k++)
        if (i + k < left) p[i + k] = from_f<T>(w[k]);
  }
}

// 4 states of B or C of one token, zeros past N
template <bool WIDE, typename T> __device__ __forceinline__ float4 load_states(const T* p, int n, int N) {
  if (WIDE) {   // N is a multiple of 4: a pack is whole or not there
    if (n >= N) return float4{0.f, 0.f, 0.f, 0.f};
    float v[4];
    load_f<4>(p + n, v);
    return float4{v[0], v[1], v[2], v[3]};
  }
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (n + 4 <= N) load_f<4, false>(p + n, v);
  else
#pragma unroll
    for (int i = 0; i < 3; i++)
      if (n + i < N) v[i] = to_f(p[n + i]);
  return float4{v[0], v[1], v[2], v[3]};
}
__device__ __forceinline__ void load_state4(const float* p, int n, int N, float (&h)[4]) {
#pragma unroll
  for (int i = 0; i < 4; i++) h[i] = n + i < N ? p[n + i] : 0.f;
}

// the thread's packs of 4 states of a tile's B, then C
template <typename T, int S, int TT, int NBC, bool WIDE>
__device__ __forceinline__ void load_bc(const ScanArgs& a, int64_t b, int g, int64_t t, int64_t t1, float4 (&o)[(NBC + NT - 1) / NT]) {
  constexpr int H = TT * S;   // packs of B
#pragma unroll
  for (int k = 0; k < (NBC + NT - 1) / NT; k++) {
    const int i = k * NT + threadIdx.x, r = i % H, n = 4 * (r % S);
    const bool in = t + r / S < t1;
    o[k] = float4{0.f, 0.f, 0.f, 0.f};
    if (i < H) {
      if (in) o[k] = load_states<WIDE>(at<T>(a.Bm, b * a.Bb + (int64_t)g * a.N + t * a.Bt, (uint32_t)(r / S * a.Bt) * sizeof(T)), n, a.N);
    } else if (i < NBC) {
      if (in) o[k] = load_states<WIDE>(at<T>(a.Cm, b * a.Cb + (int64_t)g * a.N + t * a.Ct, (uint32_t)(r / S * a.Ct) * sizeof(T)), n, a.N);
    }
  }
}

// the lane's byte of a tile's starts, and of all lanes' bytes the tile's tokens that start a sequence, a bit
// each (TT <= 32), the same in every wave
template <int TT> __device__ __forceinline__ uint32_t load_start(const ScanArgs& a, int64_t b, int64_t t, int64_t t1) {
  const int l = threadIdx.x & 63;
  return a.starts && l < TT && t + l < t1 ? *at<uint8_t>(a.starts, b * a.L + t, (uint32_t)l) : 0;
}
__device__ __forceinline__ uint32_t start_bits(uint32_t byte) { return (uint32_t)__builtin_amdgcn_ballot_w64(byte != 0); }

// Where a thread's j-th unit (16 bytes) of a row of LDS goes, r: the thread's place in the row, U: units a
// thread.  The threads' rows of units are 16 U bytes apart; the exchange of units within a thread's own
// every 256 bytes lets 8 neighbouring threads' writes of one j fall into different banks.
template <int U> __device__ __forceinline__ int unit(int r, int j) { return r * U + (j ^ (r * U >> 4 & (U - 1))); }

// Sums over the S lanes of a channel of G tokens' values, token i's left in the lanes ng with ng % G = i:
// G tokens leave by one store of all lanes (G = S up to the inner tile).  Of two tokens' values a lane
// keeps one and gives the other away.
constexpr int group_of(int S) { return S < TR ? S : TR; }
__device__ __forceinline__ float xor4(float v) { return dpp<0x1B>(dpp<SEQ_DPP_HALF_MIRROR>(v)); }   // xor 7, then xor 3
template <int S> __device__ __forceinline__ float token_sums(float (&q)[group_of(S)]) {
  const int l = threadIdx.x;
  constexpr int G = group_of(S);
  if (S == 16)
#pragma unroll
    for (int i = 0; i < G; i++) q[i] += dpp<SEQ_DPP_ROR8>(q[i]);
#pragma unroll
  for (int i = 0; 2 * i < G; i++)
    if (G > 1) q[i] = ((l & 1) ? q[2 * i + (G > 1)] : q[2 * i]) + dpp<SEQ_DPP_XOR1>((l & 1) ? q[2 * i] : q[2 * i + (G > 1)]);
#pragma unroll
  for (int i = 0; 4 * i < G; i++)
    if (G > 2) q[i] = ((l & 2) ? q[2 * i + (G > 2)] : q[2 * i]) + dpp<SEQ_DPP_XOR2>((l & 2) ? q[2 * i] : q[2 * i + (G > 2)]);
  if (G > 4) q[0] = ((l & 4) ? q[G > 4] : q[0]) + xor4((l & 4) ? q[0] : q[G > 4]);
  return q[0];
}

// STATE: the chunk's state from a zero start and its decay alone.
//
// Bound by the VALU: exp2 and 4 instructions a state and token, and what a token costs a lane beyond (3 reads of LDS, the
// sum over the channel's lanes) by its 4 states.  Bf16, 4 x 2048 x 2048 x 16: 84 us, the VALU busy in 89 % of the cycles
// (268 M states and tokens: 10.7 lane instructions each, 8 by count), the chunks' states 60 us, 93 %.  Fp32, 512 x 33 x 512
// x 16 with the states for the gradient: 74 us, 240 MB, 68 %.  Tiles whose waves share nothing, without barriers, take
// as long.
template <typename T, int S, bool STATE, bool WIDE> __global__ __launch_bounds__(NT, fwd_waves(S, sizeof(T))) void scan_fwd_kernel(ScanArgs a) {
  constexpr int TT = tile_f(S, sizeof(T)), CW = NT / S, E = TT / S, RT = CW / E, NP = 4 * S, G = group_of(S), U = E / 2;
  __shared__ float4 dd[TT][CW / 2];                                 // dt, dt u of two channels; then y in dt's place
  __shared__ float4 sB[TT][S], sC[STATE ? 1 : TT][S];
  const Where w = where<S>(a, 0, STATE ? a.nch - 1 : a.nch);
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int cl = wave * (64 / S) + lane / S, ng = lane % S;         // the lane's channel and states
  const int lt = tid / RT, lc = (tid % RT) * E;                     // the thread's part of a tile
  const int left = a.per - w.c0 - lc;                               // channels from there to the group's end
  const bool on = w.c0 + cl < a.per;
  const int mine2 = 2 * unit<U>(cl / E, cl % E / 2) + cl % 2;       // the lane's channel in a row of dd, as float2
  const int64_t t0 = (int64_t)w.chunk * a.chunk, t1 = t0 + a.chunk < a.L ? t0 + a.chunk : a.L;
  const bool z = !STATE && a.z;
  const uint32_t ou = (uint32_t)(lt * a.ut + lc) * sizeof(T), od = (uint32_t)(lt * a.dt + lc) * sizeof(T),
                 oz = (uint32_t)(lt * a.zt + lc) * sizeof(T), oo = (uint32_t)(lt * a.dim + lc) * sizeof(T);

  Raw<T, E> nu, nd, nz, cu, cz;
  constexpr int NBC = STATE ? TT * S : 2 * TT * S;                  // packs of 4 states a tile
  constexpr int PER = (NBC + NT - 1) / NT;
  float4 nbc[PER];
  uint32_t ns = 0;
  auto fetch = [&](int64_t t) {
    const int l = t + lt < t1 ? left : 0;
    ns = load_start<TT>(a, w.b, t, t1);
    load_channels<E, WIDE>(at<T>(a.u, w.b * a.ub + t * a.ut + w.ch, ou), l, nu);
    load_channels<E, WIDE>(at<T>(a.delta, w.b * a.db + t * a.dt + w.ch, od), l, nd);
    if (z) load_channels<E, WIDE>(at<T>(a.z, w.b * a.zb + t * a.zt + w.ch, oz), l, nz);
    load_bc<T, S, TT, NBC, WIDE>(a, w.b, w.g, t, t1, nbc);
  };
  float A2[4], h[4] = {0.f, 0.f, 0.f, 0.f}, dsum = 0.f;
  const int64_t ch = w.ch + (on ? cl : 0);
  load_state4(a.A + ch * a.N, 4 * ng, a.N, A2);
#pragma unroll
  for (int i = 0; i < 4; i++) A2[i] *= SEQ_LOG2E;
  if (!STATE) {
    if (a.nch > 1) load_state4(a.hin + (w.row * a.dim + ch) * NP, 4 * ng, NP, h);
    else if (a.state) load_state4(a.state + (w.b * a.dim + ch) * a.N, 4 * ng, a.N, h);
  }
  float Dv[E], bias[E];
#pragma unroll
  for (int i = 0; i < E; i++) {
    Dv[i] = !STATE && a.D && i < left ? a.D[w.ch + lc + i] : 0.f;
    bias[i] = a.bias && i < left ? a.bias[w.ch + lc + i] : 0.f;
  }
  if (t0 < t1) fetch(t0);
  for (int64_t t = t0; t < t1; t += TT) {
    const bool mine = t + lt < t1;
#pragma unroll
    for (int j = 0; j < U; j++) {
      float d[2];
#pragma unroll
      for (int k = 0; k < 2; k++) d[k] = mine && 2 * j + k < left ? softplus_f(to_f(nd.v[2 * j + k]) + bias[2 * j + k]) : 0.f;
      dd[lt][unit<U>(tid % RT, j)] = float4{d[0], d[0] * to_f(nu.v[2 * j]), d[1], d[1] * to_f(nu.v[2 * j + 1])};
    }
    cu = nu;
    cz = nz;
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int i = k * NT + tid;
      if (i < TT * S) (&sB[0][0])[i] = nbc[k];
      else if (!STATE && i < 2 * TT * S) (&sC[0][0])[i - TT * S] = nbc[k];
    }
    const uint32_t bits = start_bits(ns);
    __syncthreads();
    if (t + TT < t1) fetch(t + TT);
    // ANY: some of the n tokens start a sequence, or there are fewer than TR
    auto tokens = [&](auto any, int p, int n) {
      constexpr bool ANY = decltype(any)::value;
      float q[G] = {};
#pragma unroll
      for (int k = 0; k < TR; k++) {
        if (ANY && k >= n) break;
        const float2 d = reinterpret_cast<const float2*>(dd[p + k])[mine2];
        const float4 b = sB[p + k][ng];
        if (ANY && (bits >> (p + k) & 1)) {   // (without the product with its decay, which may be infinity: 0 times that is NaN)
          h[0] = d.y * b.x;
          h[1] = d.y * b.y;
          h[2] = d.y * b.z;
          h[3] = d.y * b.w;
          if (STATE) dsum = __builtin_nanf("");
        } else {
          h[0] = exp2_f(d.x * A2[0]) * h[0] + d.y * b.x;
          h[1] = exp2_f(d.x * A2[1]) * h[1] + d.y * b.y;
          h[2] = exp2_f(d.x * A2[2]) * h[2] + d.y * b.z;
          h[3] = exp2_f(d.x * A2[3]) * h[3] + d.y * b.w;
        }
        if (STATE) {
          dsum += d.x;
        } else {
          const float4 c = sC[p + k][ng];
          q[k % G] = c.x * h[0] + c.y * h[1] + c.z * h[2] + c.w * h[3];
          if (k % G == G - 1 || (ANY && k == n - 1)) {   // (dt of these tokens has been read by every lane of the channel)
            const float y = token_sums<S>(q);
            if (G == S || ng < G) reinterpret_cast<float2*>(dd[p + k / G * G + ng])[mine2].x = y;
          }
        }
      }
    };
    auto keep = [&](int p) {
      if (!STATE && a.ckpt && on)
        *reinterpret_cast<float4*>(a.ckpt + ((w.b * a.nck + (t + p) / TR) * a.dim + ch) * NP + 4 * ng) = float4{h[0], h[1], h[2], h[3]};
    };
    if (!bits && t + TT <= t1) {
#pragma unroll 1
      for (int p = 0; p < TT; p += TR) {
        keep(p);
        tokens(std::false_type(), p, TR);
      }
    } else {
      const int held = t1 - t < TT ? (int)(t1 - t) : TT;
#pragma unroll 1
      for (int p = 0; p < held; p += TR) {
        keep(p);
        if (bits >> p & ((1u << TR) - 1) || p + TR > held) tokens(std::true_type(), p, held - p);
        else tokens(std::false_type(), p, TR);
      }
    }
    __syncthreads();
    if (!STATE && mine) {
      float o[E];
#pragma unroll
      for (int j = 0; j < U; j++) {
        const float4 y = dd[lt][unit<U>(tid % RT, j)];
        o[2 * j] = y.x;
        o[2 * j + 1] = y.z;
      }
#pragma unroll
      for (int i = 0; i < E; i++) {
        o[i] += Dv[i] * to_f(cu.v[i]);
        const float zv = to_f(cz.v[i]);
        if (z) o[i] *= zv * sigmoid_f(zv);
      }
      store_channels<E, WIDE>(at<T>(a.out, (w.b * a.L + t) * a.dim + w.ch, oo), left, o);
    }
  }
  if (!on) return;
  if (STATE) {
    *reinterpret_cast<float4*>(a.hin + (w.row * a.dim + ch) * NP + 4 * ng) = float4{h[0], h[1], h[2], h[3]};
    if (ng == 0) a.dsum[w.row * a.dim + ch] = dsum;
  } else if (a.last && w.chunk == a.nch - 1) {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (4 * ng + i < a.N) a.last[(w.b * a.dim + ch) * a.N + 4 * ng + i] = h[i];
  }
}

// the chunks chained: what a chunk starts from takes the place of its own state.  back: from the other
// end, the gradient's way.
__global__ __launch_bounds__(NT) void scan_chain_kernel(ScanArgs a, const float* first, int NP, int back) {
  const int64_t id = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (id >= a.B * a.dim * NP) return;
  const int n = (int)(id % NP);
  const int64_t bd = id / NP, b = bd / a.dim;
  const int d = (int)(bd - b * a.dim);
  const float A2 = n < a.N ? a.A[(int64_t)d * a.N + n] * SEQ_LOG2E : 0.f;
  float h = first && n < a.N ? first[bd * a.N + n] : 0.f;
  float* p = a.hin + ((b * a.nch + (back ? a.nch - 1 : 0)) * a.dim + d) * NP + n;
  const float* q = a.dsum + (b * a.nch + (back ? a.nch - 1 : 0)) * a.dim + d;
  const int64_t stride = back ? -(int64_t)a.dim : a.dim;
  constexpr int C = 8;   // chunks whose states are loaded together
  for (int i = 0; i < a.nch; i += C, p += C * stride * NP, q += C * stride) {
    float own[C], s[C];
#pragma unroll
    for (int k = 0; k < C; k++)
      if (i + k < a.nch - 1) {   // (nothing follows the last one: its own state was not asked for)
        own[k] = p[k * stride * NP];
        s[k] = q[k * stride];
      }
#pragma unroll
    for (int k = 0; k < C; k++) {
      if (i + k >= a.nch) return;
      p[k * stride * NP] = h;
      // a start in the chunk lets nothing through, and a zero nothing of a growing state (A > 0) whose factor
      // outgrows fp32; a factor that does on its way to a product that does not: in four parts
      if (i + k < a.nch - 1) {
        const float e = exp2_f(0.25f * A2 * s[k]);
        h = s[k] == s[k] && h != 0.f ? own[k] + e * (e * (e * (e * h))) : own[k];
      }
    }
  }
}

struct ScanBwdArgs {
  ScanArgs f;
  const void* dout;
  int64_t ob, ot;
  const float* dlast;
  void *du, *ddelta, *dz, *dB, *dC;
  float *dA, *dD, *dbias, *dstate;
  float* part;    // [B * nch][dim * N + 2 dim]: dA, dD, ddelta_bias of a chunk
  float* strips;  // [sum_strips(B * nch)][dim * N + 2 dim]
  float* bc;      // [tiles][B * L][groups][2][4 S]: dB, dC of a workgroup's channels
};

// sums of v[8] over the lanes of a wave that differ in the channel (lane / S): lane l is left with
// v[4 b5 + 2 b4 + b3] of all of them (b5, b4, b3: bits of l), for S = 16 with that and the next in v[0], v[1].
// Halving: of two values a lane keeps one and gives the other away, so 8 sums over 16 lanes take 16
// instructions, not 64.
__device__ __forceinline__ float swap_add32(float x, float y) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float swap_add16(float x, float y) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int S> __device__ __forceinline__ void channel_sums(float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = swap_add32(v[i], v[i + 4]);
#pragma unroll
  for (int i = 0; i < 2; i++) v[i] = swap_add16(v[i], v[i + 2]);
  if (S < 16) {
    const bool up = threadIdx.x & 8;
    const float give = up ? v[0] : v[1], keep = up ? v[1] : v[0];
    v[0] = keep + dpp<SEQ_DPP_ROR8>(give);
  }
  if (S < 8) v[0] += xor4(v[0]);
  if (S < 4) v[0] += dpp<SEQ_DPP_XOR2>(v[0]);
  if (S < 2) v[0] += dpp<SEQ_DPP_XOR1>(v[0]);
}

// a chunk's adjoint from a zero end, and its decay: as the chunk's state, 64 us (VALU 88 %)
template <typename T, int S, bool WIDE> __global__ __launch_bounds__(NT) void scan_adjoint_kernel(ScanBwdArgs a) {
  constexpr int TT = tile_f(S, sizeof(T)), CW = NT / S, E = TT / S, RT = CW / E, NP = 4 * S, U = E / 2;
  const ScanArgs& f = a.f;
  __shared__ float4 dd[TT][CW / 2];                    // dt, dy of two channels
  __shared__ float4 sC[TT][S];
  const Where w = where<S>(f, 1, f.nch - 1);
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int cl = wave * (64 / S) + lane / S, ng = lane % S;
  const int lt = tid / RT, lc = (tid % RT) * E;
  const int left = f.per - w.c0 - lc;
  const bool on = w.c0 + cl < f.per;
  const int mine2 = 2 * unit<U>(cl / E, cl % E / 2) + cl % 2;
  const int64_t t0 = (int64_t)w.chunk * f.chunk, t1 = t0 + f.chunk < f.L ? t0 + f.chunk : f.L;
  const bool z = f.z;
  const uint32_t od = (uint32_t)(lt * f.dt + lc) * sizeof(T), oz = (uint32_t)(lt * f.zt + lc) * sizeof(T),
                 oy = (uint32_t)(lt * a.ot + lc) * sizeof(T);
  float A2[4], g[4] = {0.f, 0.f, 0.f, 0.f}, dsum = 0.f;
  const int64_t ch = w.ch + (on ? cl : 0);
  load_state4(f.A + ch * f.N, 4 * ng, f.N, A2);
#pragma unroll
  for (int i = 0; i < 4; i++) A2[i] *= SEQ_LOG2E;
  float bias[E];
#pragma unroll
  for (int i = 0; i < E; i++) bias[i] = f.bias && i < left ? f.bias[w.ch + lc + i] : 0.f;
  constexpr int NBC = TT * S, PER = (NBC + NT - 1) / NT;
  Raw<T, E> nd, nz, no;
  float4 nc[PER];
  uint32_t ns = 0;
  ScanArgs fc = f;   // C in B's place: all of it that load_bc reads
  fc.Bm = f.Cm;
  fc.Bb = f.Cb;
  fc.Bt = f.Ct;
  auto fetch = [&](int64_t t) {
    const int l = t + lt < t1 ? left : 0;
    ns = load_start<TT>(f, w.b, t, t1);
    load_channels<E, WIDE>(at<T>(f.delta, w.b * f.db + t * f.dt + w.ch, od), l, nd);
    if (z) load_channels<E, WIDE>(at<T>(f.z, w.b * f.zb + t * f.zt + w.ch, oz), l, nz);
    load_channels<E, WIDE>(at<T>(a.dout, w.b * a.ob + t * a.ot + w.ch, oy), l, no);
    load_bc<T, S, TT, NBC, WIDE>(fc, w.b, w.g, t, t1, nc);
  };
  const int64_t tiles = (t1 - t0 + TT - 1) / TT;
  if (tiles > 0) fetch(t0 + (tiles - 1) * TT);
  for (int64_t t = t0 + (tiles - 1) * TT; t >= t0; t -= TT) {
    const bool mine = t + lt < t1;
#pragma unroll
    for (int j = 0; j < U; j++) {
      float d[4];
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const int i = 2 * j + k;
        const bool in = mine && i < left;
        const float zv = to_f(nz.v[i]), ov = to_f(no.v[i]);
        d[2 * k] = in ? softplus_f(to_f(nd.v[i]) + bias[i]) : 0.f;
        d[2 * k + 1] = !in ? 0.f : z ? ov * zv * sigmoid_f(zv) : ov;
      }
      dd[lt][unit<U>(tid % RT, j)] = float4{d[0], d[1], d[2], d[3]};
    }
#pragma unroll
    for (int k = 0; k < PER; k++)
      if (k * NT + tid < NBC) (&sC[0][0])[k * NT + tid] = nc[k];
    const uint32_t bits = start_bits(ns);
    __syncthreads();
    if (t > t0) fetch(t - TT);
    auto tokens = [&](auto any, int p, int n) {
      constexpr bool ANY = decltype(any)::value;
#pragma unroll
      for (int k = TR - 1; k >= 0; k--) {
        if (ANY && k >= n) continue;
        const float2 d = reinterpret_cast<const float2*>(dd[p + k])[mine2];
        const float4 c = sC[p + k][ng];
        g[0] = exp2_f(d.x * A2[0]) * (g[0] + c.x * d.y);
        g[1] = exp2_f(d.x * A2[1]) * (g[1] + c.y * d.y);
        g[2] = exp2_f(d.x * A2[2]) * (g[2] + c.z * d.y);
        g[3] = exp2_f(d.x * A2[3]) * (g[3] + c.w * d.y);
        dsum += d.x;
        if (ANY && (bits >> (p + k) & 1)) {
          g[0] = g[1] = g[2] = g[3] = 0.f;
          dsum = __builtin_nanf("");
        }
      }
    };
    if (!bits && t + TT <= t1) {
#pragma unroll 1
      for (int p = TT - TR; p >= 0; p -= TR) tokens(std::false_type(), p, TR);
    } else {
      const int held = t1 - t < TT ? (int)(t1 - t) : TT;
#pragma unroll 1
      for (int p = (held - 1) / TR * TR; p >= 0; p -= TR) tokens(std::true_type(), p, held - p);
    }
    __syncthreads();
  }
  if (!on) return;
  *reinterpret_cast<float4*>(f.hin + (w.row * f.dim + ch) * NP + 4 * ng) = float4{g[0], g[1], g[2], g[3]};
  if (ng == 0) f.dsum[w.row * f.dim + ch] = dsum;
}

// The gradient.  An inner tile's states are walked forward again from the one that was kept (keeping all would be 8 times
// the memory traffic) and stay with their decays in registers for the way back; sums over the lanes of a channel (three a
// token) and over the channels of a wave (8 a lane) are halved at each step.  Bound by the VALU, about 26 instructions a
// state and token, at 2 waves a SIMD, which is what 8 tokens' states in registers leave (3 spill): bf16, 4 x 2048 x 2048 x
// 16, 282 us, VALU 77 %; fp32, 512 x 33 x 512 x 16, 205 us, 66 % (33 tokens are 2 tiles of 16 and one of 1).
template <typename T, int S, bool WIDE> __global__ __launch_bounds__(NT, 2) void scan_bwd_kernel(ScanBwdArgs a) {
  constexpr int TT = tile_b(S, sizeof(T)), CW = NT / S, E = TT / S, RT = CW / E, NP = 4 * S, G = group_of(S);
  const ScanArgs& f = a.f;
  __shared__ float4 dd[TT][CW];                        // dt, dy, u, dt u; then dt, dy, sum g B, sum g (a h') A
  __shared__ float yb[TT][CW];                         // sum C h
  __shared__ float4 sB[TT][S], sC[TT][S];
  __shared__ float bc[4][TT][2 * NP];
  const Where w = where<S>(f, 0, f.nch);
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int cl = wave * (64 / S) + lane / S, ng = lane % S;
  const int lt = tid / RT, lc = (tid % RT) * E;
  const int left = f.per - w.c0 - lc;
  const bool on = w.c0 + cl < f.per;
  const int mine4 = unit<E>(cl / E, cl % E);           // the lane's channel in a row of dd
  const int64_t t0 = (int64_t)w.chunk * f.chunk, t1 = t0 + f.chunk < f.L ? t0 + f.chunk : f.L;
  const bool z = f.z;
  const uint32_t ou = (uint32_t)(lt * f.ut + lc) * sizeof(T), od = (uint32_t)(lt * f.dt + lc) * sizeof(T),
                 oz = (uint32_t)(lt * f.zt + lc) * sizeof(T), oy = (uint32_t)(lt * a.ot + lc) * sizeof(T),
                 oo = (uint32_t)(lt * f.dim + lc) * sizeof(T), ok = (uint32_t)(cl * NP + 4 * ng) * 4u;

  constexpr int NBC = 2 * TT * S, PER = (NBC + NT - 1) / NT;
  Raw<T, E> nu, nd, nz, no, cu, cd, cz, co;
  float4 nbc[PER];
  uint32_t ns = 0;
  auto fetch = [&](int64_t t) {
    const int l = t + lt < t1 ? left : 0;
    ns = load_start<TT>(f, w.b, t, t1);
    load_channels<E, WIDE>(at<T>(f.u, w.b * f.ub + t * f.ut + w.ch, ou), l, nu);
    load_channels<E, WIDE>(at<T>(f.delta, w.b * f.db + t * f.dt + w.ch, od), l, nd);
    if (z) load_channels<E, WIDE>(at<T>(f.z, w.b * f.zb + t * f.zt + w.ch, oz), l, nz);
    load_channels<E, WIDE>(at<T>(a.dout, w.b * a.ob + t * a.ot + w.ch, oy), l, no);
    load_bc<T, S, TT, NBC, WIDE>(f, w.b, w.g, t, t1, nbc);
  };
  const int64_t tiles = (t1 - t0 + TT - 1) / TT;
  if (tiles > 0) fetch(t0 + (tiles - 1) * TT);   // (under way while the rest is loaded)

  float A[4], A2[4], dA[4] = {0.f, 0.f, 0.f, 0.f}, g[4] = {0.f, 0.f, 0.f, 0.f};
  const int64_t ch = w.ch + (on ? cl : 0);
  load_state4(f.A + ch * f.N, 4 * ng, f.N, A);
#pragma unroll
  for (int i = 0; i < 4; i++) A2[i] = A[i] * SEQ_LOG2E;
  if (f.nch > 1) load_state4(f.hin + (w.row * f.dim + ch) * NP, 4 * ng, NP, g);
  else if (a.dlast) load_state4(a.dlast + (w.b * f.dim + ch) * f.N, 4 * ng, f.N, g);
  float Dv[E], bias[E], dD[E] = {}, dbias[E] = {};
#pragma unroll
  for (int i = 0; i < E; i++) {
    Dv[i] = f.D && i < left ? f.D[w.ch + lc + i] : 0.f;
    bias[i] = f.bias && i < left ? f.bias[w.ch + lc + i] : 0.f;
  }
  for (int64_t t = t0 + (tiles - 1) * TT; t >= t0; t -= TT) {
    const bool mine = t + lt < t1;
#pragma unroll
    for (int i = 0; i < E; i++) {
      const bool in = mine && i < left;
      const float uv = to_f(nu.v[i]), zv = to_f(nz.v[i]), ov = to_f(no.v[i]);
      const float d = in ? softplus_f(to_f(nd.v[i]) + bias[i]) : 0.f;
      const float dy = !in ? 0.f : z ? ov * zv * sigmoid_f(zv) : ov;
      dd[lt][unit<E>(tid % RT, i)] = float4{d, dy, uv, d * uv};
    }
    cu = nu;
    cd = nd;
    cz = nz;
    co = no;
    float4 hc[TT / TR];
#pragma unroll
    for (int p = 0; p < TT / TR; p++) {
      hc[p] = float4{0.f, 0.f, 0.f, 0.f};
      if (on && t + p * TR < t1) hc[p] = *reinterpret_cast<const float4*>(at<float>(f.ckpt, ((w.b * f.nck + t / TR + p) * f.dim + w.ch) * NP, ok));
    }
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int i = k * NT + tid;
      if (i < TT * S) (&sB[0][0])[i] = nbc[k];
      else if (i < 2 * TT * S) (&sC[0][0])[i - TT * S] = nbc[k];
    }
    const uint32_t bits = start_bits(ns);
    __syncthreads();
    if (t > t0) fetch(t - TT);
    // The inner tile at p from the state h0: its states and decays forward, kept, then the adjoint back.  ANY: some
    // of the n tokens start a sequence, or there are fewer than TR.  A start's decay is 0 whatever the state (0 times
    // infinity is NaN).
    auto tokens = [&](auto any, int p, int n, const float4 h0) {
      constexpr bool ANY = decltype(any)::value;
      const uint32_t marks = bits >> p;
      float e[TR][4], h[TR + 1][4], q[G] = {};
      h[0][0] = h0.x; h[0][1] = h0.y; h[0][2] = h0.z; h[0][3] = h0.w;
#pragma unroll
      for (int k = 0; k < TR; k++) {
        if (ANY && k >= n) break;
        const float4 d = dd[p + k][mine4];
        const float4 b = sB[p + k][ng], c = sC[p + k][ng];
        const float bv[4] = {b.x, b.y, b.z, b.w}, cv[4] = {c.x, c.y, c.z, c.w};
        const bool st = ANY && (marks >> k & 1);
        float y = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          e[k][i] = exp2_f(d.x * A2[i]);
          const float ah = e[k][i] * h[k][i];
          h[k + 1][i] = (st ? 0.f : ah) + d.w * bv[i];
          y += cv[i] * h[k + 1][i];
        }
        q[k % G] = y;
        if (k % G == G - 1 || (ANY && k == n - 1)) {
          y = token_sums<S>(q);
          if (G == S || ng < G) yb[p + k / G * G + ng][cl] = y;
        }
      }
      // the tile is read again rather than held, 12 registers a token (the compiler must not see that it is the same)
      asm volatile("" : "+s"(p));
      float q1[G] = {}, q2[G] = {};
#pragma unroll
      for (int k = TR - 1; k >= 0; k--) {
        if (ANY && k >= n) continue;
        const float4 d = dd[p + k][mine4];
        const float4 b = sB[p + k][ng], c = sC[p + k][ng];
        const float bv[4] = {b.x, b.y, b.z, b.w}, cv[4] = {c.x, c.y, c.z, c.w};
        const bool st = ANY && (marks >> k & 1);
        float s1 = 0.f, s2 = 0.f, v[8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          g[i] += cv[i] * d.y;
          v[4 + i] = h[k + 1][i] * d.y;
          v[i] = g[i] * d.w;
          s1 += g[i] * bv[i];
          float ek = e[k][i];
          asm("" : "+v"(ek));   // (e h is multiplied again: kept from above it would take 4 registers a token)
          const float ah = ek * h[k][i], gah = g[i] * (st ? 0.f : ah);
          s2 += gah * A[i];
          dA[i] += gah * d.x;
          g[i] = st ? 0.f : g[i] * ek;
        }
        q1[k % G] = s1;
        q2[k % G] = s2;
        if (k % G == 0) {
          const float2 s = {token_sums<S>(q1), token_sums<S>(q2)};
          if (G == S || ng < G) *reinterpret_cast<float2*>(&dd[p + k + ng][mine4].z) = s;
        }
        channel_sums<S>(v);
        if (S >= 8 || (lane & 7) < S) {
          const int o = (lane >> 5) * NP + 4 * ng + 2 * (lane >> 4 & 1);
          if (S < 16) bc[wave][p + k][o + (lane >> 3 & 1)] = v[0];
          else {
            bc[wave][p + k][o] = v[0];
            bc[wave][p + k][o + 1] = v[1];
          }
        }
      }
    };
    const int held = t1 - t < TT ? (int)(t1 - t) : TT;
#pragma unroll
    for (int i = TT / TR - 1; i >= 0; i--) {
      if (i * TR >= held) continue;
      if (bits >> (i * TR) & ((1u << TR) - 1) || i * TR + TR > held) tokens(std::true_type(), i * TR, held - i * TR, hc[i]);
      else tokens(std::false_type(), i * TR, TR, hc[i]);
    }
    __syncthreads();
    if (mine) {
      float du[E], dr[E], dz[E];
#pragma unroll
      for (int i = 0; i < E; i++) {
        const float4 s = dd[lt][unit<E>(tid % RT, i)];
        const float dt = s.x, dy = s.y, uv = to_f(cu.v[i]);
        du[i] = Dv[i] * dy + dt * s.z;
        dr[i] = i < left ? (s.w + uv * s.z) * sigmoid_f(to_f(cd.v[i]) + bias[i]) : 0.f;
        dD[i] += dy * uv;
        dbias[i] += dr[i];
        const float zv = to_f(cz.v[i]), sg = sigmoid_f(zv);
        dz[i] = to_f(co.v[i]) * (yb[lt][lc + i] + Dv[i] * uv) * (sg * (1.f + zv * (1.f - sg)));
      }
      const int64_t o = (w.b * f.L + t) * f.dim + w.ch;
      store_channels<E, WIDE>(at<T>(a.du, o, oo), left, du);
      store_channels<E, WIDE>(at<T>(a.ddelta, o, oo), left, dr);
      if (z) store_channels<E, WIDE>(at<T>(a.dz, o, oo), left, dz);
    }
    // this workgroup's share of dB and dC
    const int64_t tile = w.c0 / CW;
    for (int i = tid; i < TT * 2 * NP; i += NT) {
      const int k = i / (2 * NP), j = i - k * 2 * NP;
      if (t + k < t1)
        a.bc[(((tile * f.B + w.b) * f.L + t + k) * f.groups + w.g) * (2 * NP) + j] = bc[0][k][j] + bc[1][k][j] + bc[2][k][j] + bc[3][k][j];
    }
  }
  float* part = a.part + w.row * ((int64_t)f.dim * (f.N + 2));
  if (on) {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (4 * ng + i < f.N) {
        part[ch * f.N + 4 * ng + i] = dA[i];
        if (a.dstate && w.chunk == 0) a.dstate[(w.b * f.dim + ch) * f.N + 4 * ng + i] = g[i];
      }
  }
  // dD and ddelta_bias: the sums of the TT threads that share channels
  __syncthreads();
#pragma unroll
  for (int i = 0; i < E; i++) *reinterpret_cast<float2*>(&dd[lt][lc + i]) = float2{dD[i], dbias[i]};
  __syncthreads();
  if (tid < CW && w.c0 + tid < f.per) {
    float2 s = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < TT; k++) {
      const float2 v = *reinterpret_cast<const float2*>(&dd[k][tid]);
      s.x += v.x;
      s.y += v.y;
    }
    part[(int64_t)f.dim * f.N + w.ch + tid] = s.x;
    part[(int64_t)f.dim * (f.N + 1) + w.ch + tid] = s.y;
  }
}

// dB, dC [B][L][groups][N] from the workgroups' shares
template <typename T> __global__ __launch_bounds__(NT) void scan_bc_kernel(const float* bc, int64_t rows, int N, int NP, int tiles, T* dB, T* dC) {
  for (int64_t id = (int64_t)blockIdx.x * NT + threadIdx.x; id < rows * 2 * NP; id += (int64_t)gridDim.x * NT) {
    const int64_t r = id / (2 * NP);
    const int j = (int)(id - r * 2 * NP), n = j % NP;
    if (n >= N) continue;
    float s = 0.f;
#pragma unroll 8
    for (int i = 0; i < tiles; i++) s += bc[i * rows * 2 * NP + id];
    (j < NP ? dB : dC)[r * N + n] = from_f<T>(s);
  }
}

// sums of 64 columns of part[rows][cols], the rows dealt to 16 waves and joined in wave order; in wave 0
__device__ __forceinline__ float rows_sum(const float* part, int64_t rows, int64_t cols, int64_t c) {
  __shared__ float sh[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
  if (c < cols) {
    int64_t r = w;
    for (; r + 48 < rows; r += 64) {
      const float* p = part + r * cols + c;
      s0 += p[0];
      s1 += p[16 * cols];
      s2 += p[32 * cols];
      s3 += p[48 * cols];
    }
    for (; r < rows; r += 16) s0 += part[r * cols + c];
  }
  sh[w][lane] = (s0 + s1) + (s2 + s3);
  __syncthreads();
  float s = 0.f;
  if (!w)
#pragma unroll
    for (int i = 0; i < 16; i++) s += sh[i][lane];
  return s;
}

// dA, dD, ddelta_bias from the chunks' rows
__global__ __launch_bounds__(1024) void scan_sums_kernel(const float* part, int64_t rows, int dim, int N, float* dA, float* dD, float* dbias) {
  const int64_t cols = (int64_t)dim * (N + 2), c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const float s = rows_sum(part, rows, cols, c);
  if (threadIdx.x >= 64 || c >= cols) return;
  const int64_t na = (int64_t)dim * N;
  if (c < na) dA[c] = s;
  else if (c < na + dim) { if (dD) dD[c - na] = s; }
  else if (dbias) dbias[c - na - dim] = s;
}
// many rows first in strips of STRIP (40944 rows of 550: by the few workgroups of all rows 540 us)
constexpr int64_t STRIP = 512;
__global__ __launch_bounds__(1024) void scan_strips_kernel(const float* part, int64_t rows, int64_t cols, float* out) {
  const int64_t c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63), r = blockIdx.y * STRIP;
  const float s = rows_sum(part + r * cols, rows - r < STRIP ? rows - r : STRIP, cols, c);
  if (threadIdx.x < 64 && c < cols) out[blockIdx.y * cols + c] = s;
}

// One token: a lane holds 4 states of a channel, a workgroup NT / S channels of one sequence (so that the
// sequence is a scalar).  Bound by the states' way from and to memory.  STREAM: states that outgrow the 256 MB
// of cache before HBM go past the caches: at 8192 x 512 x 16 (268 MB) 98 against 102 us, 113 against 127 us with
// the rest of a step's inputs; where they fit it is the other way (134 MB: 51 against 45 us).
template <typename T, int S, bool W4, bool STREAM> __global__ __launch_bounds__(NT) void scan_step_kernel(ScanArgs a) {
  typedef float V4 __attribute__((ext_vector_type(4)));
  const int ng = threadIdx.x % S;
  const int64_t n = a.B * a.tiles;
  for (int64_t at = blockIdx.x; at < n; at += gridDim.x) {
    const int64_t b = (uint64_t)at < (1ull << 32) ? (uint32_t)at / (uint32_t)a.tiles : at / a.tiles;
    const int d0 = (int)(at - b * a.tiles) * (NT / S) + threadIdx.x / S;
    const bool on = d0 < a.dim;
    const int d = on ? d0 : 0;
    const int64_t bd = b * a.dim + d;
    float h[4] = {0.f, 0.f, 0.f, 0.f}, A2[4];
    const float* hp = a.state ? a.state + bd * a.N + 4 * ng : nullptr;
    if (W4) {
      if (hp) {
        const V4 v = STREAM ? __builtin_nontemporal_load((const V4*)hp) : *(const V4*)hp;
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = v[i];
      }
      load_f<4>(a.A + (int64_t)d * a.N + 4 * ng, A2);
    } else {
      if (hp) load_state4(hp - 4 * ng, 4 * ng, a.N, h);
      load_state4(a.A + (int64_t)d * a.N, 4 * ng, a.N, A2);
    }
    const float uv = to_f(((const T*)a.u)[b * a.ub + d]);
    const float raw = to_f(((const T*)a.delta)[b * a.db + d]) + (a.bias ? a.bias[d] : 0.f);
    const float zv = a.z ? to_f(((const T*)a.z)[b * a.zb + d]) : 0.f;
    const int g = d / a.per;
    const float4 bm = load_states<W4>((const T*)a.Bm + b * a.Bb + (int64_t)g * a.N, 4 * ng, a.N);
    const float4 cm = load_states<W4>((const T*)a.Cm + b * a.Cb + (int64_t)g * a.N, 4 * ng, a.N);
    const float dt = softplus_f(raw), dtu = dt * uv;
    const bool begins = a.starts && a.starts[b];
    if (begins) h[0] = h[1] = h[2] = h[3] = 0.f;
    const float bv[4] = {bm.x, bm.y, bm.z, bm.w}, cv[4] = {cm.x, cm.y, cm.z, cm.w};
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float e = exp2_f(dt * (A2[i] * SEQ_LOG2E));
      h[i] = (begins ? 0.f : e) * h[i] + dtu * bv[i];   // (a decay may be infinity: 0 times that is NaN)
      y += cv[i] * h[i];
    }
    y = group_sum<S>(y);
    if (!on) continue;
    if (W4) {
      const V4 v = {h[0], h[1], h[2], h[3]};
      if (STREAM) __builtin_nontemporal_store(v, (V4*)(a.last + bd * a.N + 4 * ng));
      else *(V4*)(a.last + bd * a.N + 4 * ng) = v;
    } else
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (4 * ng + i < a.N) a.last[bd * a.N + 4 * ng + i] = h[i];
    if (ng == 0) {
      if (a.D) y += a.D[d] * uv;
      if (a.z) y *= zv * sigmoid_f(zv);
      ((T*)a.out)[bd] = from_f<T>(y);
    }
  }
}

// ---- host
int lanes_of(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

bool scan_ok(const pnp_scan_desc* d) {
  return d && d->B >= 0 && d->L >= 0 && d->dim > 0 && d->dim <= (1 << 24) && d->N >= 1 && d->N <= 64 && d->groups >= 1 &&
         d->dim % d->groups == 0 && type_bytes(d->type) && d->B <= ((int64_t)1 << 31) && d->L <= ((int64_t)1 << 31);
}

// How a call is cut: chunks of the length where sequences and channels alone leave the chip idle, up to 1024
// workgroups.  A chunk costs its tokens twice (about 0.18 us a token that a workgroup walks, and with two launches more
// 10 us), so the fewer the workgroups the shorter it may be; the chain over the chunks costs 0.09 us each, which
// weighs as much as the walk at 2 sqrt(L) of them.  Measured, forward and gradient, fp32, N 16, chunks of 128 at the
// least / of 64 / 32 / 16: 1 x 1000 x 64 149 / 101 / 76 / 56 us, 4 x 192 x 128 122 / - / 50 / 40; with 128 and more
// workgroups the other way: 32 x 100 x 256 (128) 79 / 79 / 81, 100 x 128 x 256 (400) 115 / - / 143 / 149.
struct Plan { int S, tiles, nch; int64_t chunk, nck, blocks; };
Plan plan(const pnp_scan_desc* d) {
  Plan p;
  p.S = lanes_of(d->N);
  const int per = d->dim / d->groups;
  p.tiles = (int)ceil_div(per, NT / p.S);
  const int64_t base = d->B * d->groups * p.tiles;
  int64_t nch = 1;
  if (base < 512) {
    nch = ceil_div(1024, base ? base : 1);
    const int64_t most = d->L / (base <= 64 ? 16 : base <= 128 ? 64 : 128);
    if (nch > most) nch = most;
    while (nch * nch > 6 * d->L) nch = nch * 15 / 16;
    if (nch < 3) nch = 1;   // (two chunks walk as many tokens one after the other as one)
  }
  p.chunk = ceil_div(d->L ? d->L : 1, nch);
  const int tt = p.chunk > 16 ? 32 : 16;   // (whole tiles, but in the shortest)
  p.chunk = ceil_div(p.chunk, tt) * tt;
  p.nch = (int)(d->L ? ceil_div(d->L, p.chunk) : 1);
  p.nck = ceil_div(d->L, TR);
  p.blocks = base * p.nch;
  return p;
}
// strips that the sums over rows are taken in first: none for few rows, at most 2^15 (the launch's second dimension)
int64_t sum_strips(int64_t rows) { return rows > 2 * STRIP && rows <= STRIP << 15 ? ceil_div(rows, STRIP) : 0; }
int64_t split_floats(const pnp_scan_desc* d, const Plan& p) {
  return p.nch > 1 ? d->B * p.nch * d->dim * (int64_t)(4 * p.S + 1) : 0;
}

ScanArgs scan_args(const pnp_scan_desc* d, const Plan& p, float* workspace) {
  ScanArgs a{};
  a.B = d->B; a.L = d->L; a.dim = d->dim; a.N = d->N; a.groups = d->groups; a.per = d->dim / d->groups;
  a.tiles = p.tiles; a.nch = p.nch; a.chunk = p.chunk; a.nck = p.nck;
  a.u = d->u; a.delta = d->delta; a.z = d->z; a.Bm = d->Bm; a.Cm = d->Cm;
  a.ub = d->u_bstride; a.ut = d->u_tstride; a.db = d->delta_bstride; a.dt = d->delta_tstride; a.zb = d->z_bstride; a.zt = d->z_tstride;
  a.Bb = d->B_bstride; a.Bt = d->B_tstride; a.Cb = d->C_bstride; a.Ct = d->C_tstride;
  a.A = d->A; a.D = d->D; a.bias = d->delta_bias; a.state = d->state; a.starts = d->starts;
  a.out = d->out; a.last = d->last_state; a.ckpt = d->ckpt;
  if (p.nch > 1) {
    a.hin = workspace;
    a.dsum = workspace + d->B * p.nch * d->dim * (int64_t)(4 * p.S);
  }
  return a;
}

// E channels of a thread start on a 16-byte boundary (or on the whole E, where that is less) in every tensor
bool even(const void* p, int64_t s1, int64_t s2, int V, int bytes) {
  return !p || (aligned_to(p, (size_t)V * bytes) && s1 % V == 0 && s2 % V == 0);
}
bool bc_even(const ScanArgs& a, int bytes) {
  return a.N % 4 == 0 && even(a.Bm, a.Bb, a.Bt, 4, bytes) && even(a.Cm, a.Cb, a.Ct, 4, bytes);
}

#define BY_LANES(S_, S, ...)                                  \
  [&]() -> int32_t {                                          \
    switch (S_) {                                             \
      case 1: { constexpr int S = 1; __VA_ARGS__; }           \
      case 2: { constexpr int S = 2; __VA_ARGS__; }           \
      case 4: { constexpr int S = 4; __VA_ARGS__; }           \
      case 8: { constexpr int S = 8; __VA_ARGS__; }           \
    }                                                         \
    constexpr int S = 16;                                     \
    __VA_ARGS__;                                              \
  }()

// (a length is cut in chunks below 512 workgroups only, of 256 / S channels each: 2^19 threads at most)
int32_t chain(const ScanArgs& a, const float* first, int S, int back, hipStream_t st) {
  const int64_t n = a.B * a.dim * 4 * S;
  hipLaunchKernelGGL(scan_chain_kernel, dim3((unsigned)ceil_div(n, NT)), dim3(NT), 0, st, a, first, 4 * S, back);
  return pnp_check_launch("scan_chain_kernel");
}

template <typename T, int S> int32_t run_scan(ScanArgs a, int64_t blocks, hipStream_t st) {
  constexpr int E = tile_f(S, sizeof(T)) / S, V = E * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : E;
  const bool wide = bc_even(a, sizeof(T)) && a.per % V == 0 && a.dim % V == 0 && even(a.u, a.ub, a.ut, V, sizeof(T)) && even(a.delta, a.db, a.dt, V, sizeof(T)) &&
           even(a.z, a.zb, a.zt, V, sizeof(T)) && even(a.out, 0, 0, V, sizeof(T));
  auto go = [&](auto w) -> int32_t {
    if (a.nch > 1) {
      hipLaunchKernelGGL((scan_fwd_kernel<T, S, true, w>), dim3((unsigned)(blocks / a.nch * (a.nch - 1))), dim3(NT), 0, st, a);
      if (const int32_t rc = pnp_check_launch("scan_fwd_kernel (chunks)")) return rc;
      if (const int32_t rc = chain(a, a.state, S, 0, st)) return rc;
    }
    hipLaunchKernelGGL((scan_fwd_kernel<T, S, false, w>), dim3((unsigned)blocks), dim3(NT), 0, st, a);
    return pnp_check_launch("scan_fwd_kernel");
  };
  return wide ? go(std::true_type()) : go(std::false_type());
}

template <typename T, int S> int32_t run_scan_bwd(ScanBwdArgs a, int64_t blocks, hipStream_t st) {
  // the wider of the two kernels' packs
  constexpr int E = tile_f(S, sizeof(T)) / S, V = E * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : E;
  ScanArgs& f = a.f;
  const bool wide = bc_even(f, sizeof(T)) && f.per % V == 0 && f.dim % V == 0 && even(f.u, f.ub, f.ut, V, sizeof(T)) && even(f.delta, f.db, f.dt, V, sizeof(T)) &&
           even(f.z, f.zb, f.zt, V, sizeof(T)) && even(a.dout, a.ob, a.ot, V, sizeof(T)) && even(a.du, 0, 0, V, sizeof(T)) &&
           even(a.ddelta, 0, 0, V, sizeof(T)) && even(a.dz, 0, 0, V, sizeof(T));
  auto go = [&](auto w) -> int32_t {
    if (f.nch > 1) {
      hipLaunchKernelGGL((scan_adjoint_kernel<T, S, w>), dim3((unsigned)(blocks / f.nch * (f.nch - 1))), dim3(NT), 0, st, a);
      if (const int32_t rc = pnp_check_launch("scan_adjoint_kernel")) return rc;
      if (const int32_t rc = chain(f, a.dlast, S, 1, st)) return rc;
    }
    hipLaunchKernelGGL((scan_bwd_kernel<T, S, w>), dim3((unsigned)blocks), dim3(NT), 0, st, a);
    return pnp_check_launch("scan_bwd_kernel");
  };
  if (const int32_t rc = wide ? go(std::true_type()) : go(std::false_type())) return rc;
  const int64_t rows = f.B * f.L * f.groups, n = ceil_div(rows * 8 * S, NT);
  if (n) {
    hipLaunchKernelGGL((scan_bc_kernel<T>), dim3((unsigned)(n < (1 << 22) ? n : (1 << 22))), dim3(NT), 0, st, a.bc, rows, f.N, 4 * S, f.tiles,
                       (T*)a.dB, (T*)a.dC);
    if (const int32_t rc = pnp_check_launch("scan_bc_kernel")) return rc;
  }
  const int64_t cols = (int64_t)f.dim * (f.N + 2), part_rows = f.B * f.nch, strips = sum_strips(part_rows);
  const float* part = a.part;
  if (strips) {
    hipLaunchKernelGGL(scan_strips_kernel, dim3((unsigned)ceil_div(cols, 64), (unsigned)strips), dim3(1024), 0, st, part, part_rows, cols, a.strips);
    if (const int32_t rc = pnp_check_launch("scan_strips_kernel")) return rc;
    part = a.strips;
  }
  hipLaunchKernelGGL(scan_sums_kernel, dim3((unsigned)ceil_div(cols, 64)), dim3(1024), 0, st, part, strips ? strips : part_rows, f.dim, f.N, a.dA,
                     a.dD, a.dbias);
  return pnp_check_launch("scan_sums_kernel");
}

template <typename T, int S> int32_t run_step(ScanArgs a, hipStream_t st) {
  const bool w4 = a.N == 4 * S && bc_even(a, sizeof(T)) && aligned_to(a.A, 16) && aligned_to(a.last, 16) && (!a.state || aligned_to(a.state, 16));
  a.tiles = (int)ceil_div(a.dim, NT / S);
  const int64_t n = a.B * a.tiles;
  const unsigned grid = (unsigned)(n < (1 << 22) ? n : (1 << 22));
  const bool stream = a.B * a.dim * a.N >= 50 * 1000 * 1000;   // 200 MB of states
  if (w4 && stream) hipLaunchKernelGGL((scan_step_kernel<T, S, true, true>), dim3(grid), dim3(NT), 0, st, a);
  else if (w4) hipLaunchKernelGGL((scan_step_kernel<T, S, true, false>), dim3(grid), dim3(NT), 0, st, a);
  else hipLaunchKernelGGL((scan_step_kernel<T, S, false, false>), dim3(grid), dim3(NT), 0, st, a);
  return pnp_check_launch("scan_step_kernel");
}

}  // namespace
}  // namespace seq

using namespace seq;

extern "C" int64_t pnp_scan_ckpt_floats(const pnp_scan_desc* d) {
  if (!scan_ok(d)) {
    pnp_set_error("pnp_scan_ckpt_floats: bad shape or type");
    return PNP_ERR_ARG;
  }
  const Plan p = plan(d);
  return d->B * p.nck * d->dim * (int64_t)(4 * p.S);
}

extern "C" int64_t pnp_scan_workspace(const pnp_scan_desc* d) {
  if (!scan_ok(d)) {
    pnp_set_error("pnp_scan_workspace: bad shape or type");
    return PNP_ERR_ARG;
  }
  return split_floats(d, plan(d));
}

// a tile's offsets are 32-bit: 32 tokens of a stride, in bytes
static bool strides_ok(const pnp_scan_desc* d) {
  for (int64_t s : {d->u_tstride, d->delta_tstride, d->z_tstride, d->B_tstride, d->C_tstride, (int64_t)d->dim})
    if (s < 0 || s > PNP_SCAN_MAX_TSTRIDE) return false;
  return true;
}

static int32_t scan_check(const pnp_scan_desc* d, const Plan& p, const char* fn) {
  if (!strides_ok(d)) {
    pnp_set_error("%s: a token stride is out of range", fn);
    return PNP_ERR_ARG;
  }
  if (!d->A || (d->B && d->L && (!d->u || !d->delta || !d->Bm || !d->Cm))) {
    pnp_set_error("%s: null buffer", fn);
    return PNP_ERR_ARG;
  }
  if (p.blocks >= (1 << 24)) {   // (a launch holds fewer than 2^32 threads)
    pnp_set_error("%s: too many sequences for one launch", fn);
    return PNP_ERR_ARG;
  }
  if (d->ckpt && d->ckpt_floats < pnp_scan_ckpt_floats(d)) {
    pnp_set_error("%s: ckpt too small", fn);
    return PNP_ERR_ARG;
  }
  if ((d->ckpt && !aligned_to(d->ckpt, 16)) || (d->workspace && !aligned_to(d->workspace, 16))) {
    pnp_set_error("%s: ckpt and workspace are aligned to 16 bytes", fn);
    return PNP_ERR_ARG;
  }
  return PNP_OK;
}

extern "C" int32_t pnp_selective_scan(const pnp_scan_desc* d, void* stream) {
  const char* fn = "pnp_selective_scan";
  if (!scan_ok(d)) {
    pnp_set_error("%s: bad shape or type", fn);
    return PNP_ERR_ARG;
  }
  if (!d->B || (!d->L && !d->last_state)) return PNP_OK;
  const Plan p = plan(d);
  if (const int32_t rc = scan_check(d, p, fn)) return rc;
  if (d->L && !d->out) {
    pnp_set_error("%s: null buffer", fn);
    return PNP_ERR_ARG;
  }
  const int64_t need = split_floats(d, p);
  if (need && (!d->workspace || d->workspace_floats < need)) {
    pnp_set_error("%s: workspace too small", fn);
    return PNP_ERR_ARG;
  }
  const ScanArgs a = scan_args(d, p, d->workspace);
  const hipStream_t st = (hipStream_t)stream;
  return SEQ_BY_TYPE(d->type, T, return BY_LANES(p.S, S, return (run_scan<T, S>(a, p.blocks, st))));
}

extern "C" int64_t pnp_scan_bwd_workspace(const pnp_scan_bwd_desc* d) {
  if (!d || !scan_ok(&d->f)) {
    pnp_set_error("pnp_scan_bwd_workspace: bad shape or type");
    return PNP_ERR_ARG;
  }
  const pnp_scan_desc& f = d->f;
  const Plan p = plan(&f);
  return split_floats(&f, p) + (f.B * p.nch + sum_strips(f.B * p.nch)) * f.dim * (int64_t)(f.N + 2) + p.tiles * f.B * f.L * f.groups * (int64_t)(8 * p.S);
}

extern "C" int32_t pnp_selective_scan_bwd(const pnp_scan_bwd_desc* d, void* stream) {
  const char* fn = "pnp_selective_scan_bwd";
  if (!d || !scan_ok(&d->f)) {
    pnp_set_error("%s: bad shape or type", fn);
    return PNP_ERR_ARG;
  }
  const pnp_scan_desc& f = d->f;
  const Plan p = plan(&f);
  if (const int32_t rc = scan_check(&f, p, fn)) return rc;
  if ((int64_t)f.dim * (f.N + 2) >= ((int64_t)1 << 28)) {
    pnp_set_error("%s: too many channels for one launch", fn);
    return PNP_ERR_ARG;
  }
  if (!d->dA || (f.B && f.L && (!f.ckpt || !d->dout || !d->du || !d->ddelta || !d->dB || !d->dC || !f.z != !d->dz))) {
    pnp_set_error("%s: null buffer", fn);
    return PNP_ERR_ARG;
  }
  if (d->dout_tstride < 0 || d->dout_tstride > PNP_SCAN_MAX_TSTRIDE) {
    pnp_set_error("%s: a token stride is out of range", fn);
    return PNP_ERR_ARG;
  }
  const int64_t need = pnp_scan_bwd_workspace(d);
  if (need && (!d->workspace || !aligned_to(d->workspace, 16) || d->workspace_floats < need)) {
    pnp_set_error("%s: workspace too small", fn);
    return PNP_ERR_ARG;
  }
  const hipStream_t st = (hipStream_t)stream;
  ScanBwdArgs a{};
  a.f = scan_args(&f, p, d->workspace);
  a.dout = d->dout; a.ob = d->dout_bstride; a.ot = d->dout_tstride; a.dlast = d->dlast;
  a.du = d->du; a.ddelta = d->ddelta; a.dz = d->dz; a.dB = d->dB; a.dC = d->dC;
  a.dA = d->dA; a.dD = d->dD; a.dbias = d->ddelta_bias; a.dstate = d->dstate;
  a.part = d->workspace + split_floats(&f, p);
  a.strips = a.part + f.B * p.nch * f.dim * (int64_t)(f.N + 2);
  a.bc = a.strips + sum_strips(f.B * p.nch) * f.dim * (int64_t)(f.N + 2);
  if (!f.B) {
    hipLaunchKernelGGL(scan_sums_kernel, dim3((unsigned)ceil_div((int64_t)f.dim * (f.N + 2), 64)), dim3(1024), 0, st, (const float*)nullptr,
                       (int64_t)0, f.dim, f.N, a.dA, a.dD, a.dbias);
    return pnp_check_launch("scan_sums_kernel");
  }
  return SEQ_BY_TYPE(f.type, T, return BY_LANES(p.S, S, return (run_scan_bwd<T, S>(a, p.blocks, st))));
}

extern "C" int32_t pnp_selective_scan_step(const pnp_scan_desc* d, void* stream) {
  const char* fn = "pnp_selective_scan_step";
  if (!scan_ok(d) || d->L != 1) {
    pnp_set_error("%s: bad shape or type", fn);
    return PNP_ERR_ARG;
  }
  if (!d->B) return PNP_OK;
  if (!d->A || !d->u || !d->delta || !d->Bm || !d->Cm || !d->out || !d->last_state) {
    pnp_set_error("%s: null buffer", fn);
    return PNP_ERR_ARG;
  }
  Plan p{};
  p.S = lanes_of(d->N);
  p.nch = 1;
  const ScanArgs a = scan_args(d, p, nullptr);
  const hipStream_t st = (hipStream_t)stream;
  return SEQ_BY_TYPE(d->type, T, return BY_LANES(p.S, S, return (run_step<T, S>(a, st))));
}
