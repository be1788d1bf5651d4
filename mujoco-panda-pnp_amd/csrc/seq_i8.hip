// seq_i8.hip — the product in 8-bit integers with a scale per token and per output channel
// (include/pnp.h pnp_matmul_i8): out[m][n] = (sum_k q[m][k] wq[n][k]) scale[m] wscale[n] + bias[n].
//
// Both operands run along k in memory, so a lane's 16 bytes of a row are its operand of
// v_mfma_i32_16x16x64_i8 as they lie (any order of k serves, as long as both operands have the same).
// The weights are the instruction's rows and the tokens its columns: a lane then holds 4 output channels
// of one token.  The channels of a wave are dealt to its fragments so that a lane's 4 of neighbouring fragments make a
// pack of V channels (16 bytes of output) and the 4 lanes of a token 4 packs in a row, whole 64 bytes a store:
// fragment i's row 4 g + r is channel 4 V (i / (V / 4)) + V g + 4 (i % (V / 4)) + r.  Against 4 WN neighbouring
// channels a lane (stores of 16 bytes with gaps between): 8192 x 8192 x 1024 109 -> 89 us, 8192 x 1024 x 256 12.8 -> 11.1.
#include <type_traits>

#include "seq_dev.h"

namespace seq {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

struct I8Args {
  int64_t M, qs, ws;
  int N, K;
  const int8_t *q, *w;
  const float *scale, *wscale, *bias;
  void* out;
  int wide;   // rows of out start on 16-byte boundaries
};

// 16 bytes of a row, wherever they lie.  (Aligned words shifted into place, one more load and 4 instructions: 8191^3
// 1014 against 732 us.)
__device__ __forceinline__ v4i whole16(const int8_t* p) {
  v4i v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
// the same from k on, zeros past the row's K: its end by the words that hold some of it, shifted into place (by bytes
// the few rows of 64 x 1000 x 1001 took 12 us)
typedef int __attribute__((may_alias)) word;
__device__ __forceinline__ v4i load16(const int8_t* row, int k, int K) {
  const int n = K - k;
  if (n >= 16) return whole16(row + k);
  v4i v = {0, 0, 0, 0};
  if (n <= 0) return v;
  const int8_t* p = row + k;
  const int by = (int)((uintptr_t)p & 3);
  const word* w = reinterpret_cast<const word*>(p - by);
  int d[5];
#pragma unroll
  for (int i = 0; i < 5; i++) d[i] = 4 * i < by + n ? w[i] : 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int left = n - 4 * i;   // bytes of word i that are the row's
    v[i] = (int)__builtin_amdgcn_alignbyte((uint32_t)d[i + 1], (uint32_t)d[i], (uint32_t)by) &
           (left >= 4 ? -1 : left <= 0 ? 0 : (1 << 8 * left) - 1);
  }
  return v;
}

// 16 bytes a lane from memory to LDS, at `lds` + 16 * lane, without registers.  Written out, since the
// compiler cannot tell the stages apart and would let every read of LDS wait for every such load: whoever
// reads what it brings waits for it (s_waitcnt vmcnt) and for the other waves (a barrier) itself.
__device__ __forceinline__ void load_to_lds(const int8_t* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// Workgroups go to the 8 XCDs in turn: each XCD gets a run of tiles of its own, and walks it in blocks of
// 8 tiles along the tokens, so that its L2 holds the rows and columns that the tiles at work share.
__device__ __forceinline__ void tile_of(int id, int tiles_n, int tiles_m, int& tn, int& tm) {
  const int total = tiles_n * tiles_m, per = total / 8, rest = total % 8;
  const int x = id % 8, k = id / 8;
  const int t = x * per + (x < rest ? x : rest) + k;   // the x-th run: the first `rest` of them have one more
  const int band = t / (8 * tiles_n), h = tiles_m - 8 * band < 8 ? tiles_m - 8 * band : 8, r = t - band * 8 * tiles_n;
  tn = r / h;
  tm = 8 * band + r % h;
}

// A lane's C channels: packs of V, 4 V apart, from n on.
template <typename T> constexpr int pack_of() { return 16 / (int)sizeof(T); }
template <typename T> __device__ __forceinline__ int channel(int n, int i) {
  constexpr int V = pack_of<T>();
  return n + i / V * 4 * V + i % V;
}
// what they are scaled by and get added
template <typename T, int C> struct Channels {
  float s[C], b[C];
  __device__ __forceinline__ Channels(const I8Args& a, int n) {
#pragma unroll
    for (int i = 0; i < C; i++) {
      const int c = channel<T>(n, i);
      s[i] = c < a.N ? a.wscale[c] : 0.f;
      b[i] = a.bias && c < a.N ? a.bias[c] : 0.f;
    }
  }
};
template <typename T, int C>
__device__ __forceinline__ void store_token(const I8Args& a, int64_t m, int n, const int (&acc)[C], const Channels<T, C>& ch) {
  if (m >= a.M) return;
  const float sm = a.scale[m];
  T* o = (T*)a.out + m * a.N;
  float f[C];
#pragma unroll
  for (int i = 0; i < C; i++) f[i] = (float)acc[i] * sm * ch.s[i] + ch.b[i];
  constexpr int V = C < pack_of<T>() ? C : pack_of<T>();
  if (a.wide) {   // N is a multiple of the pack: a pack is whole or past the end
#pragma unroll
    for (int i = 0; i < C; i += V) {
      float w[V];
#pragma unroll
      for (int k = 0; k < V; k++) w[k] = f[i + k];
      if (channel<T>(n, i) < a.N) store_f<V>(o + channel<T>(n, i), w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < C; i++)
      if (channel<T>(n, i) < a.N) o[channel<T>(n, i)] = from_f<T>(f[i]);
  }
}

constexpr int BK = 64;   // bytes of k a stage
__device__ __forceinline__ int k_of(int g) { return g == 0 ? 0 : g == 1 ? 3 : g == 2 ? 1 : 2; }

// A BN (channels) x BM (tokens) tile by WGN x WGM waves, a stage of BK bytes of k of both operands at a time
// through LDS.  A row of a stage is 4 chunks of 16 bytes; chunk c of row r lies at c ^ f(r), f the bits of r
// in which the 4 groups of a fragment's 16 rows differ (r / 4 for tokens, r / V for channels, mod 4).  LDS
// serves a 16-byte read 16 lanes at a time, of the first 32 lanes 0 .. 3, 12 .. 15, 20 .. 27 and then the others;
// with chunk k_of(g) for the lanes' g-th sixteen (any order of k serves) each such set meets 16 different bank
// groups: 2.0 -> 1.0 cycles of LDS a read against the order 0, 1, 2, 3.
//
// FAST (rows on 16-byte boundaries, K a multiple of 16): ST stages, filled by loads into LDS; such a load writes
// 64 lanes' chunks in a row, so the lane's global address carries the exchange; chunks past K come from `zeros`.  A
// stage's operands are read into registers under the product of the stage before (a quarter of a wave's registers;
// bf16 out, 8192^3 493 -> 477 us, 2048 x 2048 x 8192 50 -> 46 us, against reading them before their own product),
// and its buffer is loaded anew, ST stages on, as soon as everybody has.  Otherwise two stages, by way of
// registers that hold the next two.
//
// Bound by the matrix cores and the clock that the card's power leaves them: 8192^3 450 to 550 us from run to run, 2.4 to
// 2.0 POP/s (the library's int8 product 533 us).  They are busy in 65 % of the cycles; a wave waits in 29 % of its own,
// for LDS and at the stages' barriers.  Short sums by their output:
// 8192 x 1024 x 256 11 us, of which a launch of one tile 4.5 and the writing of 17 MB about 5.
__device__ const v4i zeros[1] = {};

template <typename T, int BM, int BN, int WGM, int WGN, bool FAST>
__global__ __launch_bounds__(64 * WGM* WGN, 2) void i8_tile_kernel(I8Args a) {
  constexpr int NT = 64 * WGM * WGN, ST = FAST ? 4 : 2, WM = BM / WGM / 16, WN = BN / WGN / 16, C = 4 * WN, V = pack_of<T>(), P = V / 4;
  constexpr int LW = BN * 4 / NT, LQ = BM * 4 / NT;   // chunks of a stage a thread
  static_assert(LW * NT == BN * 4 && LQ * NT == BM * 4 && WN % P == 0, "whole chunks a thread, whole packs a lane");
  __shared__ v4i sw[ST][BN * 4], sq[ST][BM * 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = (wave % WGN) * (BN / WGN), wm = (wave / WGN) * (BM / WGM);
  int tn, tm;
  tile_of(blockIdx.x, (a.N + BN - 1) / BN, (int)((a.M + BM - 1) / BM), tn, tm);
  const int n0 = tn * BN;
  const int64_t m0 = (int64_t)tm * BM;
  const int nk = (a.K + BK - 1) / BK;
  // the thread's rows and chunks; rows past the end are the last one's again, and their results are not stored
  const int8_t *pw[LW], *pq[LQ];
  int cw[LW], cq[LQ];
#pragma unroll
  for (int i = 0; i < LW; i++) {
    const int r = (i * NT + tid) >> 2;
    cw[i] = ((tid & 3) ^ (r / V & 3)) * 16;
    pw[i] = a.w + (int64_t)(n0 + r < a.N ? n0 + r : a.N - 1) * a.ws;
  }
#pragma unroll
  for (int i = 0; i < LQ; i++) {
    const int r = (i * NT + tid) >> 2;
    cq[i] = ((tid & 3) ^ (r >> 2 & 3)) * 16;
    pq[i] = a.q + (m0 + r < a.M ? m0 + r : a.M - 1) * a.qs;
  }
  v4i acc[WN][WM];
#pragma unroll
  for (int i = 0; i < WN; i++)
#pragma unroll
    for (int j = 0; j < WM; j++) acc[i][j] = v4i{0, 0, 0, 0};
  const int fr = lane & 15, fc = lane >> 4, kc = k_of(fc);
  struct Operands { v4i w[WN], q[WM]; };
  auto read = [&](int buf, Operands& f) {
#pragma unroll
    for (int i = 0; i < WN; i++) {
      const int r = wn + i / P * 4 * V + (fr >> 2) * V + i % P * 4 + (fr & 3);
      f.w[i] = sw[buf][r * 4 + (kc ^ (r / V & 3))];
    }
#pragma unroll
    for (int j = 0; j < WM; j++) {
      const int r = wm + j * 16 + fr;
      f.q[j] = sq[buf][r * 4 + (kc ^ (r >> 2 & 3))];
    }
  };
  auto product = [&](const Operands& f) {
#pragma unroll
    for (int j = 0; j < WM; j++)
#pragma unroll
      for (int i = 0; i < WN; i++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.w[i], f.q[j], acc[i][j], 0, 0, 0);
  };
  if constexpr (FAST) {
    const uint32_t lw = lds_address(&sw[0][wave * 64]), lq = lds_address(&sq[0][wave * 64]);
    auto fetch = [&](int s) {   // stage s; past the last one: zeros that nobody reads, so that every wave counts the same loads
      const int buf = s % ST, k = s * BK;
#pragma unroll
      for (int i = 0; i < LW; i++)
        load_to_lds(k + cw[i] < a.K ? pw[i] + k + cw[i] : (const int8_t*)zeros, lw + (buf * BN * 4 + i * NT) * 16);
#pragma unroll
      for (int i = 0; i < LQ; i++)
        load_to_lds(k + cq[i] < a.K ? pq[i] + k + cq[i] : (const int8_t*)zeros, lq + (buf * BM * 4 + i * NT) * 16);
    };
    // before stage s's product: this wave's loads of stage s + 1 have arrived, and what it read of stage s is in
    // registers; then, past the barrier, everybody's have and is: the buffer of stage s is free
    auto meet = [&]() {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((ST - 2) * (LW + LQ)) : "memory");
      __builtin_amdgcn_s_barrier();
    };
    Operands f0, f1;
#pragma unroll
    for (int s = 0; s < ST - 1; s++) fetch(s);
    meet();
    fetch(ST - 1);
    read(0, f0);
    for (int s = 0; s < nk; s += 2) {
      meet();
      fetch(s + ST);
      read((s + 1) % ST, f1);
      product(f0);
      meet();
      fetch(s + ST + 1);
      read((s + 2) % ST, f0);
      if (s + 1 < nk) product(f1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no load into LDS outlives the workgroup
  } else {
    struct Chunks { v4i w[LW], q[LQ]; } r0, r1;
    auto fetch = [&](int s, Chunks& r) {
      if ((s + 1) * BK <= a.K) {
#pragma unroll
        for (int i = 0; i < LW; i++) r.w[i] = whole16(pw[i] + s * BK + cw[i]);
#pragma unroll
        for (int i = 0; i < LQ; i++) r.q[i] = whole16(pq[i] + s * BK + cq[i]);
      } else {
#pragma unroll
        for (int i = 0; i < LW; i++) r.w[i] = load16(pw[i], s * BK + cw[i], a.K);
#pragma unroll
        for (int i = 0; i < LQ; i++) r.q[i] = load16(pq[i], s * BK + cq[i], a.K);
      }
    };
    auto put = [&](int buf, const Chunks& r) {
#pragma unroll
      for (int i = 0; i < LW; i++) sw[buf][i * NT + tid] = r.w[i];
#pragma unroll
      for (int i = 0; i < LQ; i++) sq[buf][i * NT + tid] = r.q[i];
    };
    auto stage = [&](int s, Chunks& r) {   // r: stage s + 1, and then s + 3
      Operands f;
      __syncthreads();   // stage s is there, and everybody has read stage s - 1
      read(s & 1, f);
      product(f);
      put((s + 1) & 1, r);
      if (s + 3 < nk) fetch(s + 3, r);
    };
    fetch(0, r0);
    if (nk > 1) fetch(1, r1);
    put(0, r0);
    if (nk > 2) fetch(2, r0);
    for (int s = 0; s < nk; s += 2) {
      stage(s, r1);
      if (s + 1 < nk) stage(s + 1, r0);
    }
  }
  const int n = n0 + wn + fc * V;
  const Channels<T, C> ch(a, n);
#pragma unroll
  for (int j = 0; j < WM; j++) {
    int o[C];
#pragma unroll
    for (int i = 0; i < WN; i++)
#pragma unroll
      for (int r = 0; r < 4; r++) o[4 * i + r] = acc[i][j][r];
    store_token<T, C>(a, m0 + wm + j * 16 + fr, n, o, ch);
  }
}

// Few tokens (16 MT at most): the weights' bytes are what counts.  A workgroup has 16 channels, its 4 waves stages of k
// in turn, straight from memory to registers; their sums meet in LDS.  A wave takes two stages that lie together, whole
// lines of the weights (by single stages, half lines: one token by 4096 x 4096 10.7 against 7.4 us, 64 tokens 25 against
// 15).  One token by 1000 x 512 5 us and by 4096 x 4096 7.0, of which a launch in a row of them 4.5; by 16384 x 8192
// 24 us, 5.6 TB/s.  16, 33 and 64 tokens by 4096 x 4096 7.8, 13 and 15 us: N / 16 workgroups are one a CU, and each wave
// waits for its own loads.
template <typename T, int MT> __global__ __launch_bounds__(256) void i8_rows_kernel(I8Args a) {
  __shared__ v4i part[3][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fc = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int8_t* w = a.w + (int64_t)(n0 + fr < a.N ? n0 + fr : a.N - 1) * a.ws;
  const int8_t* q[MT];
#pragma unroll
  for (int j = 0; j < MT; j++) q[j] = a.q + (j * 16 + fr < a.M ? j * 16 + fr : a.M - 1) * a.qs;
  v4i acc[MT];
#pragma unroll
  for (int j = 0; j < MT; j++) acc[j] = v4i{0, 0, 0, 0};
  // a wave's two stages lie together: 4 lanes on 128 bytes of a row.  Whole ones first, then the end.
  int k = 2 * wave * BK;
  const int c = 2 * fc * 16;
#pragma unroll 4
  for (; k + 2 * BK <= a.K; k += 8 * BK) {
    const v4i f0 = whole16(w + k + c), f1 = whole16(w + k + c + 16);
#pragma unroll
    for (int j = 0; j < MT; j++) {
      acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f0, whole16(q[j] + k + c), acc[j], 0, 0, 0);
      acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f1, whole16(q[j] + k + c + 16), acc[j], 0, 0, 0);
    }
  }
  if (k < a.K) {
    const v4i f0 = load16(w, k + c, a.K), f1 = load16(w, k + c + 16, a.K);
#pragma unroll
    for (int j = 0; j < MT; j++) {
      acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f0, load16(q[j], k + c, a.K), acc[j], 0, 0, 0);
      acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f1, load16(q[j], k + c + 16, a.K), acc[j], 0, 0, 0);
    }
  }
  if (wave)
#pragma unroll
    for (int j = 0; j < MT; j++) part[wave - 1][j][lane] = acc[j];
  __syncthreads();
  if (wave) return;
  const Channels<T, 4> ch(a, n0 + fc * 4);
#pragma unroll
  for (int j = 0; j < MT; j++) {
    const v4i s = acc[j] + part[0][j][lane] + part[1][j][lane] + part[2][j][lane];
    const int o[4] = {s[0], s[1], s[2], s[3]};
    store_token<T, 4>(a, j * 16 + fr, n0 + fc * 4, o, ch);
  }
}

// ---- host
template <typename T, int BM, int BN, int WGM, int WGN> int32_t launch_tile(const I8Args& a, bool fast, hipStream_t st) {
  const dim3 grid((unsigned)(ceil_div(a.M, BM) * ceil_div(a.N, BN))), block(64 * WGM * WGN);
  if (fast) hipLaunchKernelGGL((i8_tile_kernel<T, BM, BN, WGM, WGN, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((i8_tile_kernel<T, BM, BN, WGM, WGN, false>), grid, block, 0, st, a);
  return pnp_check_launch("i8_tile_kernel");
}

template <typename T> int32_t run_i8(I8Args a, hipStream_t st) {
  a.wide = a.N % (16 / (int)sizeof(T)) == 0 && aligned_to(a.out, 16);
  const bool fast = a.K % 16 == 0 && a.qs % 16 == 0 && a.ws % 16 == 0 && aligned_to(a.q, 16) && aligned_to(a.w, 16);
  const dim3 rows((unsigned)ceil_div(a.N, 16)), block(256);
  if (a.M <= 16) hipLaunchKernelGGL((i8_rows_kernel<T, 1>), rows, block, 0, st, a);
  else if (a.M <= 32) hipLaunchKernelGGL((i8_rows_kernel<T, 2>), rows, block, 0, st, a);
  else if (a.M <= 64) hipLaunchKernelGGL((i8_rows_kernel<T, 4>), rows, block, 0, st, a);
  if (a.M <= 64) return pnp_check_launch("i8_rows_kernel");
  // the largest tile that still gives most of the 256 CUs one
  const auto tiles = [&](int b) { return ceil_div(a.M, b) * ceil_div(a.N, b); };
  if (tiles(256) >= 192) return launch_tile<T, 256, 256, 2, 4>(a, fast, st);
  if (tiles(128) >= 192) return launch_tile<T, 128, 128, 2, 2>(a, fast, st);
  return launch_tile<T, 64, 64, 2, 2>(a, fast, st);
}

}  // namespace
}  // namespace seq

using namespace seq;

extern "C" int32_t pnp_matmul_i8(const pnp_i8_desc* d, void* stream) {
  const char* fn = "pnp_matmul_i8";
  // 131071 * 128 * 128 < 2^31
  if (!d || d->M < 0 || d->M > ((int64_t)1 << 31) || d->N <= 0 || d->N > (1 << 24) || d->K <= 0 || d->K > 131071 ||
      !type_bytes(d->out_type) || d->q_stride < d->K || d->wq_stride < d->K) {
    pnp_set_error("%s: bad shape or type", fn);
    return PNP_ERR_ARG;
  }
  // a launch holds fewer than 2^32 threads: 512 a tile of 256 x 256, which is what so many outputs go by (the smaller
  // tiles serve below 192 of these, the kernel for few tokens at most N / 16 workgroups of 256)
  if (d->M > 64 && ceil_div(d->M, 256) * ceil_div(d->N, 256) >= ((int64_t)1 << 23)) {
    pnp_set_error("%s: too many tiles for one launch", fn);
    return PNP_ERR_ARG;
  }
  if (!d->M) return PNP_OK;
  if (!d->q || !d->wq || !d->scale || !d->wscale || !d->out) {
    pnp_set_error("%s: null buffer", fn);
    return PNP_ERR_ARG;
  }
  I8Args a{d->M, d->q_stride, d->wq_stride, d->N, d->K, d->q, d->wq, d->scale, d->wscale, d->bias, d->out, 0};
  const hipStream_t st = (hipStream_t)stream;
  return SEQ_BY_TYPE(d->out_type, T, return run_i8<T>(a, st));
}
