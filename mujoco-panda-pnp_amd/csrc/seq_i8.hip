// seq_i8.hip — the product in 8-bit integers with a scale per token and per output channel
// (include/pnp.h pnp_matmul_i8): out[m][n] = (sum_k q[m][k] wq[n][k]) scale[m] wscale[n] + bias[n].
//
// Both operands run along k in memory, so a lane's 16 bytes of a row are its operand of
// v_mfma_i32_16x16x64_i8 as they lie (any order of k serves, as long as both operands have the same).
// The weights are the instruction's rows and the tokens its columns: a lane then holds 4 neighbouring
// output channels of one token and stores them together.
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
};

// 16 bytes of a row from k on, zeros past its K elements; any alignment
__device__ __forceinline__ v4i load16(const int8_t* row, int k, int K) {
  v4i v = {0, 0, 0, 0};
  if (k + 16 <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else if (k < K) {
    int w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; i++)
      if (k + i < K) w[i >> 2] |= (int)(uint8_t)row[k + i] << (8 * (i & 3));
    v = v4i{w[0], w[1], w[2], w[3]};
  }
  return v;
}

// 4 neighbouring channels of one token
template <typename T> __device__ __forceinline__ void store4(const I8Args& a, int64_t m, int n, v4i acc) {
  if (m >= a.M) return;
  const float sm = a.scale[m];
  T* o = (T*)a.out + m * a.N + n;
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    f[i] = 0.f;
    if (n + i < a.N) f[i] = (float)acc[i] * sm * a.wscale[n + i] + (a.bias ? a.bias[n + i] : 0.f);
  }
  if (n + 4 <= a.N && (a.N & 3) == 0) {
    store_f<4>(o, f);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (n + i < a.N) o[i] = from_f<T>(f[i]);
  }
}

// A BN (channels) x BM (tokens) tile by 4 waves, 2 x 2, 128 bytes of k at a time through LDS.
// A row of the tile is 128 bytes, 8 chunks; chunk c of row r lies at c ^ (r / 2 % 8), so the 16 rows
// that a fragment's 16 lanes read lie in 16 different bank groups.
template <typename T, int BM, int BN> __global__ __launch_bounds__(256) void i8_tile_kernel(I8Args a) {
  constexpr int WM = BM / 2 / 16, WN = BN / 2 / 16;
  __shared__ v4i sw[BN * 8], sq[BM * 8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wn = (wave & 1) * (BN / 2), wm = (wave >> 1) * (BM / 2);
  const int n0 = blockIdx.x * BN;
  const int64_t m0 = (int64_t)blockIdx.y * BM;
  v4i acc[WN][WM];
#pragma unroll
  for (int i = 0; i < WN; i++)
#pragma unroll
    for (int j = 0; j < WM; j++) acc[i][j] = v4i{0, 0, 0, 0};
  for (int k0 = 0; k0 < a.K; k0 += 128) {
#pragma unroll
    for (int i = 0; i < BN * 8 / 256; i++) {
      const int s = i * 256 + tid, r = s >> 3, c = (s & 7) ^ ((r >> 1) & 7);
      const int n = n0 + r < a.N ? n0 + r : a.N - 1;
      sw[s] = load16(a.w + n * a.ws, k0 + c * 16, a.K);
    }
#pragma unroll
    for (int i = 0; i < BM * 8 / 256; i++) {
      const int s = i * 256 + tid, r = s >> 3, c = (s & 7) ^ ((r >> 1) & 7);
      const int64_t m = m0 + r < a.M ? m0 + r : a.M - 1;
      sq[s] = load16(a.q + m * a.qs, k0 + c * 16, a.K);
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 2; kk++) {
      v4i fw[WN], fq[WM];
      const int c = kk * 4 + (lane >> 4);
#pragma unroll
      for (int i = 0; i < WN; i++) {
        const int r = wn + i * 16 + (lane & 15);
        fw[i] = sw[r * 8 + (c ^ ((r >> 1) & 7))];
      }
#pragma unroll
      for (int j = 0; j < WM; j++) {
        const int r = wm + j * 16 + (lane & 15);
        fq[j] = sq[r * 8 + (c ^ ((r >> 1) & 7))];
      }
#pragma unroll
      for (int i = 0; i < WN; i++)
#pragma unroll
        for (int j = 0; j < WM; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], fq[j], acc[i][j], 0, 0, 0);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < WN; i++)
#pragma unroll
    for (int j = 0; j < WM; j++)
      store4<T>(a, m0 + wm + j * 16 + (lane & 15), n0 + wn + i * 16 + (lane >> 4) * 4, acc[i][j]);
}

template <typename T> int32_t run_i8(const I8Args& a, hipStream_t st) {
  constexpr int BM = 128, BN = 128;
  const dim3 grid((unsigned)ceil_div(a.N, BN), (unsigned)ceil_div(a.M, BM));
  hipLaunchKernelGGL((i8_tile_kernel<T, BM, BN>), grid, dim3(256), 0, st, a);
  return pnp_check_launch("i8_tile_kernel");
}

}  // namespace
}  // namespace seq

using namespace seq;

extern "C" int32_t pnp_matmul_i8(const pnp_i8_desc* d, void* stream) {
  const char* fn = "pnp_matmul_i8";
  // 65535 * 64 tokens: a grid's second dimension; 131071 * 127 * 127 < 2^31
  if (!d || d->M < 0 || d->M > 65535 * (int64_t)64 || d->N <= 0 || d->N > (1 << 24) || d->K <= 0 || d->K > 131071 ||
      !type_bytes(d->out_type) || d->q_stride < d->K || d->wq_stride < d->K) {
    pnp_set_error("%s: bad shape or type", fn);
    return PNP_ERR_ARG;
  }
  if (!d->M) return PNP_OK;
  if (!d->q || !d->wq || !d->scale || !d->wscale || !d->out) {
    pnp_set_error("%s: null buffer", fn);
    return PNP_ERR_ARG;
  }
  I8Args a{d->M, d->q_stride, d->wq_stride, d->N, d->K, d->q, d->wq, d->scale, d->wscale, d->bias, d->out};
  const hipStream_t st = (hipStream_t)stream;
  return SEQ_BY_TYPE(d->out_type, T, return run_i8<T>(a, st));
}
