// Operators that end in 8 bits in front of a linear layer, and their backward passes (sm_100a).
//
//   row_quant_kernel<OP_NORM>  h = T(x + r), y = h * rsqrt(mean h^2 + eps) * w, codes = Q(y)
//   row_quant_kernel<OP_GATE>  y = g * sigma(g) * u,                            codes = Q(y)
//   row_quant_kernel<OP_COPY>  y = x,                                           codes = Q(y)
//   rms_norm_backward_kernel, column_sum_kernel, silu_mul_backward_kernel
//
// Q is either the block format of the FP8 linear layer (E4M3 codes, one power of two for each 32/64/128 columns,
// the rule of tcfp_quantize) or int8 with one float scale for each row.  y stays in 32 bits between the operator
// and the rounding to 8: nothing is rounded to 16 bits on the way.
#include "common.cuh"
#include "launch.h"

namespace tcfp {
namespace {

enum { OP_NORM = 0, OP_GATE = 1, OP_COPY = 2 };

constexpr int kMaxWarps = 32;
constexpr int kMaxNormWidth = 32768;     // a row's values stay in the registers of 1024 threads
constexpr int kMaxGateWidth = 1 << 26;   // column indices in 32 bits, column blocks in gridDim.y

struct RowParams {
  const void* a;          // x, or gate
  const void* b;          // residual (nullable), or up
  int64_t lda, ldb;
  const void* w;
  int w_bf16;
  float eps;
  void* h;                // x + residual (nullable)
  float* rstd;            // nullable
  uint8_t* codes;
  int64_t ldc;
  void* scale;            // int8 plane (width / block, rows), or float (rows)
  uint8_t* sf;            // nullable
  __nv_bfloat16* deq;     // nullable
  int64_t rows;
  int width;
  int block;
};

// ---- eight values of a row ----------------------------------------------------
// VEC: eight neighbours, 16-byte accesses.  Otherwise eight values a whole row of threads apart, so that neighbouring
// threads still touch neighbouring values.
template <bool BF16>
__device__ __forceinline__ float load1(const void* base, int64_t i) {
  if constexpr (BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[i]);
  else return reinterpret_cast<const float*>(base)[i];
}
template <bool BF16>
__device__ __forceinline__ void store1(void* base, int64_t i, float v) {
  if constexpr (BF16) reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<float*>(base)[i] = v;
}

template <bool BF16, bool VEC>
__device__ __forceinline__ void load8(float (&v)[8], const void* base, int64_t row_start, int i0, int step, int width) {
  if constexpr (VEC) {
    if (i0 >= width) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    } else if constexpr (BF16) {
      const uint4 raw = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(base) + row_start + i0);
      const uint32_t wd[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(wd[j] << 16);
        v[2 * j + 1] = __uint_as_float(wd[j] & 0xFFFF0000u);
      }
    } else {
      const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + row_start + i0);
      const float4 lo = p[0], hi = p[1];
      v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
      v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (i0 + j * step < width) ? load1<BF16>(base, row_start + i0 + j * step) : 0.f;
  }
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&p);
}

template <bool BF16, bool VEC>
__device__ __forceinline__ void store8(const float (&v)[8], void* base, int64_t row_start, int i0, int step, int width) {
  if constexpr (VEC) {
    if (i0 >= width) return;
    if constexpr (BF16) {
      *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(base) + row_start + i0) =
          make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    } else {
      float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + row_start + i0);
      p[0] = make_float4(v[0], v[1], v[2], v[3]);
      p[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j * step < width) store1<BF16>(base, row_start + i0 + j * step, v[j]);
  }
}

// ---- reductions over the threads of one row --------------------------------------
// maximum that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <bool MAX>
__device__ __forceinline__ float warp_reduce(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float other = __shfl_xor_sync(0xFFFFFFFFu, v, o);
    v = MAX ? max_nan(v, other) : v + other;
  }
  return v;
}
// blockDim.x threads (a multiple of 32) share a row; slots: kMaxWarps floats of shared memory for each row of the block,
// not used for anything else in the meantime.  The order is fixed.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* slots) {
  v = warp_reduce<MAX>(v);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  float* s = slots + threadIdx.y * warps;
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_reduce<MAX>(lane < warps ? s[lane] : 0.f);
}

// ---- int8 with one scale for each row ----------------------------------------------
// code = round_half_even(y / s) with the quotient rounded to 32 bits.  y * (1/s) is off by less than 3e-5 of a step, so
// the division itself is only needed where the product falls that near to the middle between two codes.
__device__ __forceinline__ int int8_code(float y, float s, float inv_s) {
  const float q = y * inv_s;
  float r = rintf(q);
  if (fabsf(fabsf(q - r) - 0.5f) < 1e-4f) r = rintf(__fdiv_rn(y, s));
  return __float2int_rn(r);
}

// ---- the operators ------------------------------------------------------------------
// silu(g) * u.  __expf and the fast division are good to a few units in the last place of 32 bits (and give the
// limits 0 and g for large |g|); the result is rounded to 8 bits.
__device__ __forceinline__ float gated(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// the value in front of the row statistics: the stream h, the gated activation, or x itself
template <int OP, bool BF16, bool VEC>
__device__ __forceinline__ void load_value(float (&v)[8], const RowParams& p, int64_t row, int i0, int step) {
  load8<BF16, VEC>(v, p.a, row * p.lda, i0, step, p.width);
  if constexpr (OP != OP_COPY) {
    if (OP == OP_NORM && p.b == nullptr) return;
    float o[8];
    load8<BF16, VEC>(o, p.b, row * p.ldb, i0, step, p.width);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (OP == OP_GATE) {
        v[j] = gated(v[j], o[j]);
      } else {
        // the stream is kept in the inputs' type and the statistics are those of what is kept
        v[j] = v[j] + o[j];
        if constexpr (BF16) v[j] = __bfloat162float(__float2bfloat16_rn(v[j]));
      }
    }
  }
}

template <bool VEC>
__device__ __forceinline__ void apply_weight(float (&v)[8], const RowParams& p, float rstd, int i0, int step) {
  float w[8];
  if (p.w_bf16) load8<true, VEC>(w, p.w, 0, i0, step, p.width);
  else load8<false, VEC>(w, p.w, 0, i0, step, p.width);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = v[j] * rstd * w[j];
}

template <bool VEC>
__device__ __forceinline__ void store_int8(const float (&v)[8], const RowParams& p, int64_t row, int i0, int step, float s,
                                           float inv_s) {
  int c[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = int8_code(v[j], s, inv_s);
  if constexpr (VEC) {
    if (i0 < p.width) {
      uint32_t wd[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        wd[k] = (uint32_t)(c[4 * k] & 0xFF) | ((uint32_t)(c[4 * k + 1] & 0xFF) << 8) |
                ((uint32_t)(c[4 * k + 2] & 0xFF) << 16) | ((uint32_t)c[4 * k + 3] << 24);
      *reinterpret_cast<uint2*>(p.codes + row * p.ldc + i0) = make_uint2(wd[0], wd[1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j * step < p.width) p.codes[row * p.ldc + i0 + j * step] = (uint8_t)c[j];
  }
  if (p.deq != nullptr) {
    float d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = (float)c[j] * s;
    store8<true, VEC>(d, p.deq, row * (int64_t)p.width, i0, step, p.width);
  }
}

// E4M3 codes of eight neighbours; block / 8 neighbouring lanes share an exponent
__device__ __forceinline__ void store_block(const float (&v)[8], const RowParams& p, int64_t row, int i0, bool live) {
  float am = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) am = fmaxf(am, fabsf(v[j]));
  const int group = p.block >> 3;
  for (int o = 1; o < group; o <<= 1) am = fmaxf(am, __shfl_xor_sync(0xFFFFFFFFu, am, o));
  if (!live || i0 >= p.width) return;
  const int e = block_exponent_fast<false>(am);
  const float fwd = exp2_int(-e), inv = exp2_int(e);
  uint32_t pc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) pc[j] = encode_fp8x2<false>(v[2 * j] * fwd, v[2 * j + 1] * fwd);
  *reinterpret_cast<uint2*>(p.codes + row * p.ldc + i0) = make_uint2(pc[0] | (pc[1] << 16), pc[2] | (pc[3] << 16));
  if (p.deq != nullptr) {
    uint32_t d[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = decode_fp8x2<false>(pc[j]);
      d[j] = pack_bf16(f.x * inv, f.y * inv);
    }
    *reinterpret_cast<uint4*>(p.deq + row * (int64_t)p.width + i0) = make_uint4(d[0], d[1], d[2], d[3]);
  }
  if (i0 % p.block == 0) {
    const int64_t num_kb = p.width / p.block, kb = i0 / p.block;
    reinterpret_cast<int8_t*>(p.scale)[kb * p.rows + row] = (int8_t)e;
    if (p.sf != nullptr) {
      const int64_t k_groups = (num_kb + 3) >> 2;
      p.sf[sf_chunk_offset(row, kb, k_groups)] = e8m0_from_exp(e);
      // the last chunk is filled up with 2^0
      if (kb == num_kb - 1)
        for (int64_t k = num_kb; k < 4 * k_groups; ++k) p.sf[sf_chunk_offset(row, k, k_groups)] = 127;
    }
  }
}

// blockDim = (threads of a row, rows of the block).  A thread holds 8 * NC values of its row in registers; NC = 0 walks
// a row of any width and loads it again for each pass.  gridDim.y > 1 (only where no statistic spans the row) splits the
// row's columns.
template <int OP, bool BF16, bool VEC, bool BLOCK, int NC>
__global__ void __launch_bounds__(NC == 1 || NC == 2 ? 512 : 1024) row_quant_kernel(const RowParams p) {
  __shared__ float s_sum[kMaxWarps], s_max[kMaxWarps];
  const int T = blockDim.x;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < p.rows;
  const int64_t r = live ? row : p.rows - 1;
  const int step = T;
  const int span = 8 * T;
  const int first = (VEC ? 8 : 1) * (int)threadIdx.x + (NC ? NC : 1) * span * (int)blockIdx.y;
  const int chunks = NC ? NC : (p.width + span - 1) / span;
  float v[NC ? NC : 1][8];

  float rstd = 1.f;
  if constexpr (OP == OP_NORM) {
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < chunks; ++c) {
      float (&x)[8] = v[NC ? c : 0];
      load_value<OP, BF16, VEC>(x, p, r, first + c * span, step);
      if (live && p.h != nullptr) store8<BF16, VEC>(x, p.h, r * (int64_t)p.width, first + c * span, step, p.width);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(x[j], x[j], sum);
    }
    sum = row_reduce<false>(sum, s_sum);
    rstd = rsqrtf(sum / (float)p.width + p.eps);
    if (live && p.rstd != nullptr && threadIdx.x == 0) p.rstd[r] = rstd;
  }
  // from here on the values that are rounded to 8 bits
  auto value = [&](int c) {
    float (&x)[8] = v[NC ? c : 0];
    if (OP != OP_NORM || NC == 0) load_value<OP, BF16, VEC>(x, p, r, first + c * span, step);
    if constexpr (OP == OP_NORM) apply_weight<VEC>(x, p, rstd, first + c * span, step);
  };
  if constexpr (BLOCK) {
#pragma unroll
    for (int c = 0; c < chunks; ++c) {
      value(c);
      store_block(v[NC ? c : 0], p, r, first + c * span, live);
    }
  } else {
    float am = 0.f;
#pragma unroll
    for (int c = 0; c < chunks; ++c) {
      value(c);
#pragma unroll
      for (int j = 0; j < 8; ++j) am = max_nan(am, fabsf(v[NC ? c : 0][j]));
    }
    am = row_reduce<true>(am, s_max);
    const float s = __fdiv_rn(am < kAmaxFloor ? kAmaxFloor : am, 127.f);
    const float inv_s = __frcp_rn(s);
    if (live && threadIdx.x == 0) reinterpret_cast<float*>(p.scale)[r] = s;
#pragma unroll
    for (int c = 0; c < chunks; ++c) {
      if constexpr (NC == 0) value(c);
      if (live) store_int8<VEC>(v[NC ? c : 0], p, r, first + c * span, step, s, inv_s);
    }
  }
}

// ---- backward of the norm ------------------------------------------------------------
struct NormBwdParams {
  const void *dy, *h, *dh;      // dh: gradient of the stream itself (nullable)
  int64_t ld_dy, ld_h, ld_dh;
  const float* rstd;
  const void* w;
  int w_bf16;
  void* dx;
  float* dw;                    // (gridDim.x, width) partial sums
  int64_t rows;
  int width;
};

// dx = rstd * (g - hat * mean(g * hat)) + dh with g = dy * w, hat = h * rstd;  dw = sum over rows of dy * hat.
// A block walks the rows blockIdx.x, blockIdx.x + gridDim.x, ...; a thread owns the same 8 * NC columns of all of
// them and keeps their part of dw in registers.
template <bool BF16, bool VEC, int NC>
__global__ void __launch_bounds__(1024) rms_norm_backward_kernel(const NormBwdParams p) {
  __shared__ float slots[2][kMaxWarps];
  const int step = blockDim.x, span = 8 * step;
  const int first = (VEC ? 8 : 1) * (int)threadIdx.x;
  float acc[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[c][j] = 0.f;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const float rstd = __ldg(p.rstd + row);
    float g[NC][8], hat[NC][8];
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i0 = first + c * span;
      load8<BF16, VEC>(g[c], p.dy, row * p.ld_dy, i0, step, p.width);
      load8<BF16, VEC>(hat[c], p.h, row * p.ld_h, i0, step, p.width);
      float w[8];
      if (p.w_bf16) load8<true, VEC>(w, p.w, 0, i0, step, p.width);
      else load8<false, VEC>(w, p.w, 0, i0, step, p.width);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        hat[c][j] *= rstd;
        acc[c][j] = fmaf(g[c][j], hat[c][j], acc[c][j]);
        g[c][j] *= w[j];
        sum = fmaf(g[c][j], hat[c][j], sum);
      }
    }
    // two sets of slots: the next row writes the other one while slower warps still read this one
    const float mean = row_reduce<false>(sum, slots[turn]) / (float)p.width;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i0 = first + c * span;
      float d[8];
      if (p.dh != nullptr) {
        load8<BF16, VEC>(d, p.dh, row * p.ld_dh, i0, step, p.width);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = fmaf(rstd, g[c][j] - hat[c][j] * mean, d[j]);
      store8<BF16, VEC>(d, p.dx, row * (int64_t)p.width, i0, step, p.width);
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c)
    store8<false, VEC>(acc[c], p.dw, (int64_t)blockIdx.x * p.width, first + c * span, step, p.width);
}

// out[c] = sum over r of partial[r, c]; 32 columns a block, the rows dealt to 8 warps and joined in a fixed order
__global__ void column_sum_kernel(const float* __restrict__ partial, int rows, int width, float* __restrict__ out) {
  __shared__ float s[8][32];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float t = 0.f;
  if (c < width)
    for (int r = threadIdx.y; r < rows; r += 8) t += partial[(int64_t)r * width + c];
  s[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.y == 0 && c < width) {
#pragma unroll
    for (int k = 1; k < 8; ++k) t += s[k][threadIdx.x];
    out[c] = t;
  }
}

// ---- backward of the gated activation ------------------------------------------------
struct GateBwdParams {
  const void *dy, *gate, *up;
  int64_t ld_dy, ld_gate, ld_up;
  void *dgate, *dup;
  int64_t ld_dgate, ld_dup;
  int64_t rows;
  int width;
};

// sigma = 1/(1+e^-g): dgate = dy * u * sigma * (1 + g (1 - sigma)), dup = dy * g * sigma
template <bool BF16, bool VEC>
__global__ void silu_mul_backward_kernel(const GateBwdParams p) {
  const int step = blockDim.x;
  const int i0 = (VEC ? 8 : 1) * (int)threadIdx.x + 8 * step * (int)blockIdx.y;
  const int64_t row = blockIdx.x;
  float d[8], g[8], u[8];
  load8<BF16, VEC>(d, p.dy, row * p.ld_dy, i0, step, p.width);
  load8<BF16, VEC>(g, p.gate, row * p.ld_gate, i0, step, p.width);
  load8<BF16, VEC>(u, p.up, row * p.ld_up, i0, step, p.width);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float sig = __fdividef(1.f, 1.f + __expf(-g[j]));
    const float ds = d[j] * sig;
    const float dg = ds * u[j] * fmaf(g[j], 1.f - sig, 1.f);
    u[j] = ds * g[j];
    g[j] = dg;
  }
  store8<BF16, VEC>(g, p.dgate, row * p.ld_dgate, i0, step, p.width);
  store8<BF16, VEC>(u, p.dup, row * p.ld_dup, i0, step, p.width);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
bool aligned16(const void* ptr, int64_t ld, int elem) {
  return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0 && ((ld * elem) & 15) == 0;
}

int round32(int x) { return (x + 31) & ~31; }

template <int OP, bool BF16, bool VEC, bool BLOCK>
int launch_row(const RowParams& p, cudaStream_t stream) {
  const int units = (p.width + 7) / 8;
  int nc, threads, rows_per_block = 1, col_blocks = 1;
  if (OP != OP_NORM && BLOCK) {
    nc = 1;
    threads = units < 256 ? round32(units) : 256;
    col_blocks = (units + threads - 1) / threads;
  } else {
    nc = units <= 512 ? 1 : units <= 1024 ? 2 : units <= 4096 ? 4 : 0;
    threads = nc ? round32((units + nc - 1) / nc) : 1024;
  }
  if (threads <= 128) rows_per_block = 256 / threads;
  if (rows_per_block > p.rows) rows_per_block = (int)p.rows;
  const dim3 grid((unsigned)((p.rows + rows_per_block - 1) / rows_per_block), (unsigned)col_blocks);
  const dim3 block((unsigned)threads, (unsigned)rows_per_block);
  if (nc == 1) row_quant_kernel<OP, BF16, VEC, BLOCK, 1><<<grid, block, 0, stream>>>(p);
  if constexpr (OP == OP_NORM || !BLOCK) {
    if (nc == 2) row_quant_kernel<OP, BF16, VEC, BLOCK, 2><<<grid, block, 0, stream>>>(p);
    if (nc == 4) row_quant_kernel<OP, BF16, VEC, BLOCK, 4><<<grid, block, 0, stream>>>(p);
  }
  if constexpr (OP != OP_NORM && !BLOCK)
    if (nc == 0) row_quant_kernel<OP, BF16, VEC, BLOCK, 0><<<grid, block, 0, stream>>>(p);
  CUDA_TRY(cudaGetLastError());
  return TCFP_OK;
}

// checks common to the three operators; `what` names the entry point
int check_row(const char* what, const RowParams& p, int dtype, int elem) {
  if (dtype != TCFP_F32 && dtype != TCFP_BF16) return fail(TCFP_ERR_INVALID, "%s: dtype %d", what, dtype);
  if (!p.a || !p.codes || !p.scale) return fail(TCFP_ERR_INVALID, "%s: NULL argument", what);
  if (p.rows < 1 || p.rows > 0x7FFFFFFF) return fail(TCFP_ERR_INVALID, "%s: rows %lld", what, (long long)p.rows);
  if (p.width < 1) return fail(TCFP_ERR_INVALID, "%s: width %d", what, p.width);
  if (p.ldc < p.width) return fail(TCFP_ERR_INVALID, "%s: ld_codes %lld is below the width %d", what, (long long)p.ldc, p.width);
  if (p.block != 0) {
    if (p.block != 32 && p.block != 64 && p.block != 128) return fail(TCFP_ERR_INVALID, "%s: block_size %d", what, p.block);
    if (p.width % p.block) return fail(TCFP_ERR_INVALID, "%s: width %d is not a multiple of block_size %d", what, p.width, p.block);
    if (p.ldc != p.width) return fail(TCFP_ERR_INVALID, "%s: block codes are dense", what);
    if (!aligned16(p.a, p.lda, elem) || (p.b && !aligned16(p.b, p.ldb, elem)) || !aligned16(p.codes, p.ldc, 1) ||
        (p.w && !aligned16(p.w, 0, 1)) || (p.h && !aligned16(p.h, 0, 1)) || (p.deq && !aligned16(p.deq, 0, 1)))
      return fail(TCFP_ERR_INVALID, "%s: the block format needs 16-byte aligned rows", what);
  } else if (p.sf) {
    return fail(TCFP_ERR_INVALID, "%s: sf_out belongs to the block format", what);
  }
  return TCFP_OK;
}

template <int OP, bool BF16>
int dispatch_row(const RowParams& p, cudaStream_t stream) {
  const int e = BF16 ? 2 : 4;
  if constexpr (OP != OP_COPY)
    if (p.block) return launch_row<OP, BF16, true, true>(p, stream);
  const bool vec = p.width % 8 == 0 && aligned16(p.a, p.lda, e) && (!p.b || aligned16(p.b, p.ldb, e)) &&
                   (!p.w || aligned16(p.w, 0, 1)) && (!p.h || aligned16(p.h, 0, 1)) && (!p.deq || aligned16(p.deq, 0, 1)) &&
                   (reinterpret_cast<uintptr_t>(p.codes) & 7u) == 0 && p.ldc % 8 == 0;
  return vec ? launch_row<OP, BF16, true, false>(p, stream) : launch_row<OP, BF16, false, false>(p, stream);
}

template <bool BF16, bool VEC>
int launch_norm_bwd(const NormBwdParams& p, int blocks, cudaStream_t stream) {
  const int units = (p.width + 7) / 8;
  const int nc = units <= 1024 ? 1 : units <= 2048 ? 2 : 4;
  const int threads = round32((units + nc - 1) / nc);
  if (nc == 1) rms_norm_backward_kernel<BF16, VEC, 1><<<blocks, threads, 0, stream>>>(p);
  else if (nc == 2) rms_norm_backward_kernel<BF16, VEC, 2><<<blocks, threads, 0, stream>>>(p);
  else rms_norm_backward_kernel<BF16, VEC, 4><<<blocks, threads, 0, stream>>>(p);
  CUDA_TRY(cudaGetLastError());
  return TCFP_OK;
}


int norm_bwd_blocks(int64_t rows) {
  const int64_t most = 4 * (int64_t)sm_count();
  return (int)(rows < most ? rows : most);
}

}  // namespace
}  // namespace tcfp

using namespace tcfp;

extern "C" int32_t tcfp_add_rms_norm_quantize(const void* x, int64_t ld_x, const void* residual, int64_t ld_residual,
                                              int32_t dtype, const void* weight, int32_t w_dtype, float eps, void* h_out,
                                              float* rstd_out, uint8_t* codes, int64_t ld_codes, void* scale_out,
                                              uint8_t* sf_out, void* deq_bf16_out, int64_t rows, int64_t width,
                                              int32_t block_size, void* stream) {
  if (width > kMaxNormWidth) return fail(TCFP_ERR_UNSUPPORTED, "tcfp_add_rms_norm_quantize: width %lld above %d", (long long)width, kMaxNormWidth);
  if (!weight) return fail(TCFP_ERR_INVALID, "tcfp_add_rms_norm_quantize: NULL weight");
  if (w_dtype != TCFP_F32 && w_dtype != TCFP_BF16) return fail(TCFP_ERR_INVALID, "tcfp_add_rms_norm_quantize: weight dtype %d", w_dtype);
  if (residual && !h_out) return fail(TCFP_ERR_INVALID, "tcfp_add_rms_norm_quantize: a residual needs h_out");
  RowParams p{x, residual, ld_x, ld_residual, weight, w_dtype == TCFP_BF16, eps, h_out, rstd_out, codes, ld_codes, scale_out,
              sf_out, reinterpret_cast<__nv_bfloat16*>(deq_bf16_out), rows, (int)width, block_size};
  const int rc = check_row("tcfp_add_rms_norm_quantize", p, dtype, dtype == TCFP_BF16 ? 2 : 4);
  if (rc != TCFP_OK) return rc;
  return dtype == TCFP_BF16 ? dispatch_row<OP_NORM, true>(p, (cudaStream_t)stream) : dispatch_row<OP_NORM, false>(p, (cudaStream_t)stream);
}

extern "C" int32_t tcfp_silu_mul_quantize(const void* gate, int64_t ld_gate, const void* up, int64_t ld_up, int32_t dtype,
                                          uint8_t* codes, int64_t ld_codes, void* scale_out, uint8_t* sf_out,
                                          void* deq_bf16_out, int64_t rows, int64_t width, int32_t block_size, void* stream) {
  if (!up) return fail(TCFP_ERR_INVALID, "tcfp_silu_mul_quantize: NULL argument");
  if (width > kMaxGateWidth) return fail(TCFP_ERR_UNSUPPORTED, "tcfp_silu_mul_quantize: width %lld", (long long)width);
  RowParams p{gate, up, ld_gate, ld_up, nullptr, 0, 0.f, nullptr, nullptr, codes, ld_codes, scale_out, sf_out,
              reinterpret_cast<__nv_bfloat16*>(deq_bf16_out), rows, (int)width, block_size};
  const int rc = check_row("tcfp_silu_mul_quantize", p, dtype, dtype == TCFP_BF16 ? 2 : 4);
  if (rc != TCFP_OK) return rc;
  return dtype == TCFP_BF16 ? dispatch_row<OP_GATE, true>(p, (cudaStream_t)stream) : dispatch_row<OP_GATE, false>(p, (cudaStream_t)stream);
}

extern "C" int32_t tcfp_int8_quantize_rows(const void* x, int64_t ld_x, int32_t dtype, uint8_t* codes, int64_t ld_codes,
                                           float* scale_out, void* deq_bf16_out, int64_t rows, int64_t width, void* stream) {
  if (width > kMaxGateWidth) return fail(TCFP_ERR_UNSUPPORTED, "tcfp_int8_quantize_rows: width %lld", (long long)width);
  RowParams p{x, nullptr, ld_x, 0, nullptr, 0, 0.f, nullptr, nullptr, codes, ld_codes, scale_out, nullptr,
              reinterpret_cast<__nv_bfloat16*>(deq_bf16_out), rows, (int)width, 0};
  const int rc = check_row("tcfp_int8_quantize_rows", p, dtype, dtype == TCFP_BF16 ? 2 : 4);
  if (rc != TCFP_OK) return rc;
  return dtype == TCFP_BF16 ? dispatch_row<OP_COPY, true>(p, (cudaStream_t)stream) : dispatch_row<OP_COPY, false>(p, (cudaStream_t)stream);
}

extern "C" size_t tcfp_rms_norm_backward_workspace_bytes(int64_t rows, int64_t width) {
  if (rows < 1 || width < 1 || width > kMaxNormWidth) return 0;
  return (size_t)norm_bwd_blocks(rows) * (size_t)width * sizeof(float);
}

extern "C" int32_t tcfp_rms_norm_backward(const void* dy, int64_t ld_dy, const void* h, int64_t ld_h, const float* rstd,
                                          int32_t dtype, const void* weight, int32_t w_dtype, const void* dh, int64_t ld_dh,
                                          void* dx, float* dw, void* workspace, int64_t rows, int64_t width, void* stream_) {
  const char* what = "tcfp_rms_norm_backward";
  cudaStream_t stream = (cudaStream_t)stream_;
  if (!dy || !h || !rstd || !weight || !dx || !dw || !workspace) return fail(TCFP_ERR_INVALID, "%s: NULL argument", what);
  if ((dtype != TCFP_F32 && dtype != TCFP_BF16) || (w_dtype != TCFP_F32 && w_dtype != TCFP_BF16))
    return fail(TCFP_ERR_INVALID, "%s: dtype %d, weight dtype %d", what, dtype, w_dtype);
  if (rows < 1 || width < 1) return fail(TCFP_ERR_INVALID, "%s: %lld rows, width %lld", what, (long long)rows, (long long)width);
  if (width > kMaxNormWidth) return fail(TCFP_ERR_UNSUPPORTED, "%s: width %lld above %d", what, (long long)width, kMaxNormWidth);
  const int e = dtype == TCFP_BF16 ? 2 : 4;
  const int blocks = norm_bwd_blocks(rows);
  NormBwdParams p{dy, h, dh, ld_dy, ld_h, ld_dh, rstd, weight, w_dtype == TCFP_BF16, dx,
                  blocks == 1 ? dw : reinterpret_cast<float*>(workspace), rows, (int)width};
  const bool vec = width % 8 == 0 && aligned16(dy, ld_dy, e) && aligned16(h, ld_h, e) && (!dh || aligned16(dh, ld_dh, e)) &&
                   aligned16(weight, 0, 1) && aligned16(dx, 0, 1) && aligned16(p.dw, 0, 1);
  int rc;
  if (dtype == TCFP_BF16) rc = vec ? launch_norm_bwd<true, true>(p, blocks, stream) : launch_norm_bwd<true, false>(p, blocks, stream);
  else rc = vec ? launch_norm_bwd<false, true>(p, blocks, stream) : launch_norm_bwd<false, false>(p, blocks, stream);
  if (rc != TCFP_OK || blocks == 1) return rc;
  column_sum_kernel<<<(unsigned)((width + 31) / 32), dim3(32, 8), 0, stream>>>(p.dw, blocks, (int)width, dw);
  CUDA_TRY(cudaGetLastError());
  return TCFP_OK;
}

extern "C" int32_t tcfp_silu_mul_backward(const void* dy, int64_t ld_dy, const void* gate, int64_t ld_gate, const void* up,
                                          int64_t ld_up, int32_t dtype, void* dgate, int64_t ld_dgate, void* dup,
                                          int64_t ld_dup, int64_t rows, int64_t width, void* stream_) {
  const char* what = "tcfp_silu_mul_backward";
  cudaStream_t stream = (cudaStream_t)stream_;
  if (!dy || !gate || !up || !dgate || !dup) return fail(TCFP_ERR_INVALID, "%s: NULL argument", what);
  if (dtype != TCFP_F32 && dtype != TCFP_BF16) return fail(TCFP_ERR_INVALID, "%s: dtype %d", what, dtype);
  if (rows < 1 || rows > 0x7FFFFFFF || width < 1 || width > kMaxGateWidth)
    return fail(TCFP_ERR_INVALID, "%s: %lld rows, width %lld", what, (long long)rows, (long long)width);
  const int e = dtype == TCFP_BF16 ? 2 : 4;
  const GateBwdParams p{dy, gate, up, ld_dy, ld_gate, ld_up, dgate, dup, ld_dgate, ld_dup, rows, (int)width};
  const bool vec = width % 8 == 0 && aligned16(dy, ld_dy, e) && aligned16(gate, ld_gate, e) && aligned16(up, ld_up, e) &&
                   aligned16(dgate, ld_dgate, e) && aligned16(dup, ld_dup, e);
  const int units = (int)((width + 7) / 8);
  const int threads = units < 256 ? round32(units) : 256;
  const dim3 grid((unsigned)rows, (unsigned)((units + threads - 1) / threads));
  if (dtype == TCFP_BF16) {
    if (vec) silu_mul_backward_kernel<true, true><<<grid, threads, 0, stream>>>(p);
    else silu_mul_backward_kernel<true, false><<<grid, threads, 0, stream>>>(p);
  } else {
    if (vec) silu_mul_backward_kernel<false, true><<<grid, threads, 0, stream>>>(p);
    else silu_mul_backward_kernel<false, false><<<grid, threads, 0, stream>>>(p);
  }
  CUDA_TRY(cudaGetLastError());
  return TCFP_OK;
}
