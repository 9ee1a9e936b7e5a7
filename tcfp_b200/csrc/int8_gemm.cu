// int8 product with a scale for each token and each channel (sm_100a).
//
//   out[m,n] = (sum_k a[m,k] b[n,k]) * s_a[m] * s_b[n] + bias[n]
//
// The sum is an exact 32-bit integer; the two scales are constant along k, so they are applied once to the finished sum.
#include "common.cuh"
#include "launch.h"

namespace tcfp {
namespace {

struct Int8Params {
  const int8_t *a, *b;
  int64_t lda, ldb;
  const float *s_a, *s_b, *bias;
  void* out;
  int M, N, K;
};

constexpr int kTile = 64;
constexpr int kStep = 64;   // bytes of K staged at a time

// 64 x 64 outputs a block of 256 threads, 4 x 4 a thread, dp4a on words staged in shared memory
template <bool OUT_BF16>
__global__ void __launch_bounds__(256) int8_gemm_kernel(const Int8Params p) {
  __shared__ int s_a[kTile][kStep / 4 + 1], s_b[kTile][kStep / 4 + 1];
  const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
  const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += kStep) {
    for (int i = threadIdx.x; i < kTile * kStep / 4; i += 256) {
      const int r = i / (kStep / 4), c = i % (kStep / 4);
      uint32_t wa = 0, wb = 0;
      for (int j = 0; j < 4; ++j) {
        const int k = k0 + 4 * c + j;
        if (k < p.K && m0 + r < p.M) wa |= (uint32_t)(uint8_t)p.a[(m0 + r) * p.lda + k] << (8 * j);
        if (k < p.K && n0 + r < p.N) wb |= (uint32_t)(uint8_t)p.b[(n0 + r) * p.ldb + k] << (8 * j);
      }
      s_a[r][c] = (int)wa;
      s_b[r][c] = (int)wb;
    }
    __syncthreads();
    for (int c = 0; c < kStep / 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(s_a[tm + 16 * i][c], s_b[tn + 16 * j][c], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + tm + 16 * i, n = n0 + tn + 16 * j;
      if (m >= p.M || n >= p.N) continue;
      float v = (float)acc[i][j] * p.s_a[m] * p.s_b[n];
      if (p.bias) v += p.bias[n];
      const int64_t at = (int64_t)m * p.N + n;
      if (OUT_BF16) reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
      else reinterpret_cast<float*>(p.out)[at] = v;
    }
}

constexpr int64_t kMaxK = 131071;   // 128 * 128 * K stays below 2^31

}  // namespace
}  // namespace tcfp

using namespace tcfp;

extern "C" int32_t tcfp_int8_gemm(const int8_t* a, int64_t ld_a, const float* s_a, const int8_t* b, int64_t ld_b,
                                  const float* s_b, const float* bias, void* out, int32_t out_dtype, int64_t M, int64_t N,
                                  int64_t K, void* stream) {
  const char* what = "tcfp_int8_gemm";
  if (!a || !b || !s_a || !s_b || !out) return fail(TCFP_ERR_INVALID, "%s: NULL argument", what);
  if (out_dtype != TCFP_F32 && out_dtype != TCFP_BF16) return fail(TCFP_ERR_INVALID, "%s: out dtype %d", what, out_dtype);
  if (M < 1 || N < 1 || K < 1 || M > (1 << 30) || N > (1 << 30))
    return fail(TCFP_ERR_INVALID, "%s: M %lld, N %lld, K %lld", what, (long long)M, (long long)N, (long long)K);
  if (K > kMaxK) return fail(TCFP_ERR_UNSUPPORTED, "%s: K %lld above %lld could overflow the integer sum", what, (long long)K, (long long)kMaxK);
  if (ld_a < K || ld_b < K || ld_a % 16 || ld_b % 16 || (reinterpret_cast<uintptr_t>(a) & 15u) || (reinterpret_cast<uintptr_t>(b) & 15u))
    return fail(TCFP_ERR_INVALID, "%s: rows of a and b start on 16-byte boundaries, ld >= K", what);
  const Int8Params p{a, b, ld_a, ld_b, s_a, s_b, bias, out, (int)M, (int)N, (int)K};
  if ((M + kTile - 1) / kTile > 65535) return fail(TCFP_ERR_UNSUPPORTED, "%s: M %lld", what, (long long)M);
  const dim3 grid((unsigned)((N + kTile - 1) / kTile), (unsigned)((M + kTile - 1) / kTile));
  if (out_dtype == TCFP_BF16) int8_gemm_kernel<true><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  else int8_gemm_kernel<false><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  CUDA_TRY(cudaGetLastError());
  return TCFP_OK;
}
