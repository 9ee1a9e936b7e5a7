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
#include <type_traits>
#include "launch.h"

namespace tcfp {
namespace {

enum { OP_NORM = 0, OP_GATE = 1, OP_COPY = 2 };

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
  int block, block_shift;
  float inv_width;
};

// ---- eight values of a row ----------------------------------------------------
// A thread's chunk of a row: VEC eight neighbours, 16-byte accesses; otherwise eight values a whole row of threads apart
// (`step`), so that neighbouring threads still touch neighbouring values.  `p` points at the chunk's first value, `left`
// values of the row lie there and behind it (none or less: nothing is touched).
template <bool BF16>
using Elem = typename std::conditional<BF16, __nv_bfloat16, float>::type;

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&p);
}

// As they come from memory, so that a load ahead holds half the registers where they are bf16.
template <bool BF16, bool VEC>
struct Raw {
  uint32_t w[BF16 && VEC ? 4 : 8];

  __device__ __forceinline__ void load(const Elem<BF16>* p, int left, int step) {
    if constexpr (VEC) {
      uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
      if (left > 0) {
        lo = reinterpret_cast<const uint4*>(p)[0];
        if constexpr (!BF16) hi = reinterpret_cast<const uint4*>(p)[1];
      }
      w[0] = lo.x; w[1] = lo.y; w[2] = lo.z; w[3] = lo.w;
      if constexpr (!BF16) { w[4] = hi.x; w[5] = hi.y; w[6] = hi.z; w[7] = hi.w; }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = j * step < left ? __float_as_uint((float)p[j * step]) : 0u;
    }
  }
  __device__ __forceinline__ void store(Elem<BF16>* p, int left, int step) const {
    if constexpr (VEC) {
      if (left <= 0) return;
      reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
      if constexpr (!BF16) reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j * step < left) p[j * step] = (Elem<BF16>)__uint_as_float(w[j]);
    }
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (BF16 && VEC) return __uint_as_float((j & 1) ? (w[j >> 1] & 0xFFFF0000u) : (w[j >> 1] << 16));
    else return __uint_as_float(w[j]);
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    if constexpr (BF16 && VEC) {
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = pack_bf16(v[2 * k], v[2 * k + 1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(v[j]);
    }
  }
};

template <bool BF16, bool VEC>
__device__ __forceinline__ void load8(float (&v)[8], const void* base, int64_t at, int left, int step) {
  Raw<BF16, VEC> r;
  r.load(reinterpret_cast<const Elem<BF16>*>(base) + at, left, step);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = r.get(j);
}
template <bool BF16, bool VEC>
__device__ __forceinline__ void store8(const float (&v)[8], void* base, int64_t at, int left, int step) {
  Raw<BF16, VEC> r;
  r.set(v);
  r.store(reinterpret_cast<Elem<BF16>*>(base) + at, left, step);
}

// ---- reductions over the threads of one row --------------------------------------
// maximum that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// over the 32 or 16 lanes that share a row
template <bool MAX>
__device__ __forceinline__ float warp_reduce(float v) {
  // numbers without a sign order as their bits do, and a NaN comes last
  if (MAX && blockDim.x >= 32) return __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(v)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (o == 16 && blockDim.x < 32) continue;
    const float other = __shfl_xor_sync(0xFFFFFFFFu, v, o);
    v = MAX ? max_nan(v, other) : v + other;
  }
  return v;
}
// Slots for the warps' parts of the rows side by side in a block.  Two sets, taken in turn: a warp may write the next
// row's while a slower one reads this row's.
struct Slots {
  float v[2][64];
};
// blockDim.x threads (16 or a multiple of 32) share a row.  Up to 8 warps: everybody adds up the row's 8 slots (those of absent
// warps hold 0); more warps have the block to themselves and join by shuffles.  The order is fixed.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* slots) {
  v = warp_reduce<MAX>(v);
  const int warps = blockDim.x >> 5;
  if (warps <= 1) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* s = slots + threadIdx.y * 8;
  if (lane == 0) s[warp] = v;
  __syncthreads();
  if (warps > 8) return warp_reduce<MAX>(lane < warps ? s[lane] : 0.f);
  const float4 a = *reinterpret_cast<const float4*>(s), b = *reinterpret_cast<const float4*>(s + 4);
  if constexpr (MAX) return max_nan(max_nan(max_nan(a.x, a.y), max_nan(a.z, a.w)), max_nan(max_nan(b.x, b.y), max_nan(b.z, b.w)));
  else return ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
}

// ---- the operators ------------------------------------------------------------------
// sigma(g) = 1 / (1 + 2^(-g log2 e)) by the approximate instructions that flush what is below 2^-126: good to about |g| + 8
// units of 2^-24 (the product's rounding becomes the exponent's error), with the limits 0 and 1 for large |g|.  For outputs of
// 8 or 16 bits, whose rounding is a thousand times that.
__device__ __forceinline__ float sigmoid(float g) {
  float t, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(g * -1.44269504f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + t));
  return r;
}
// The same good to 6 units of 2^-24 for every g, for outputs that stay in 32 bits.
__device__ __forceinline__ float sigmoid_f32(float g) { return __frcp_rn(1.f + expf(-g)); }
__device__ __forceinline__ float gated(float g, float u) { return g * sigmoid(g) * u; }

// eight values of the one or two inputs of a row
template <int OP, bool BF16, bool VEC>
struct Inputs {
  Raw<BF16, VEC> a, b;

  __device__ __forceinline__ void load(const Elem<BF16>* pa, const Elem<BF16>* pb, int left, int step) {
    a.load(pa, left, step);
    if (OP == OP_GATE || (OP == OP_NORM && pb != nullptr)) b.load(pb, left, step);
  }
  // OP_NORM: a becomes the stream x + residual as it is kept, in the inputs' type; the statistics are those of what is
  // kept.  The sum is rounded to 32 bits and then to the type, as torch adds.
  __device__ __forceinline__ void add() {
    float h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      h[j] = a.get(j) + b.get(j);
      if constexpr (BF16 && !VEC) h[j] = __bfloat162float(__float2bfloat16_rn(h[j]));
    }
    a.set(h);
  }
  // the value in front of the row statistics: the stream, the gated activation, or x itself
  __device__ __forceinline__ void value(float (&v)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = OP == OP_GATE ? gated(a.get(j), b.get(j)) : a.get(j);
  }
};

// ---- int8 with one scale for each row ----------------------------------------------
// a row that holds a NaN or an infinity has no scale
__device__ __forceinline__ float row_scale(float am) {
  return am <= 3.4028235e38f ? __fdiv_rn(fmaxf(am, kAmaxFloor), 127.f) : __uint_as_float(0x7FC00000u);
}

// code = round_half_even(y * (1/s)), reciprocal and product rounded to 32 bits: |y| <= 127.00001 s.  Adding 1.5 * 2^23 rounds
// half to even and leaves the code in the low byte.
template <bool VEC>
__device__ __forceinline__ void store_int8(const float (&v)[8], uint8_t* codes, __nv_bfloat16* deq, int left, int step, float s,
                                           float inv_s) {
  constexpr float kMagic = 12582912.f;
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = __fadd_rn(__fmul_rn(v[j], inv_s), kMagic);
  if constexpr (VEC) {
    if (left > 0) {
      uint32_t wd[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        wd[k] = __byte_perm(__byte_perm(__float_as_uint(q[4 * k]), __float_as_uint(q[4 * k + 1]), 0x0040),
                            __byte_perm(__float_as_uint(q[4 * k + 2]), __float_as_uint(q[4 * k + 3]), 0x0040), 0x5410);
      *reinterpret_cast<uint2*>(codes) = make_uint2(wd[0], wd[1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j * step < left) codes[j * step] = (uint8_t)(__float_as_uint(q[j]) & 0xFFu);
  }
  if (deq != nullptr) {
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = (q[j] - kMagic) * s;
    store8<true, VEC>(q, deq, 0, left, step);
  }
}

// E4M3 codes of eight neighbours; block / 8 neighbouring lanes share an exponent.  Returns it.
__device__ __forceinline__ int store_block(const float (&v)[8], uint8_t* codes, __nv_bfloat16* deq, int left, int block) {
  float am = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) am = fmaxf(am, fabsf(v[j]));
  am = fmaxf(am, __shfl_xor_sync(0xFFFFFFFFu, am, 1));
  am = fmaxf(am, __shfl_xor_sync(0xFFFFFFFFu, am, 2));
  if (block >= 64) am = fmaxf(am, __shfl_xor_sync(0xFFFFFFFFu, am, 4));
  if (block == 128) am = fmaxf(am, __shfl_xor_sync(0xFFFFFFFFu, am, 8));
  // the rule of block_exponent(): ceil(log2(am / 448)) with 448 = 1.75 * 2^8, so one is added from a mantissa of 1.75 on; the
  // 256 numbers there take the full rule.  am >= 1e-12, so -48 <= e <= 120 and both powers are normal numbers
  am = fmaxf(am, kAmaxFloor);
  const uint32_t up = __float_as_uint(am) + 0x200000u;
  int e = (int)(up >> 23) - 127 - 8;
  if ((up & 0x7FFFFFu) < 256u) e = block_exponent(am, kE4M3Max);
  const float fwd = __uint_as_float((uint32_t)(127 - e) << 23), inv = __uint_as_float((uint32_t)(127 + e) << 23);
  uint32_t pc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) pc[j] = encode_fp8x2<false>(v[2 * j] * fwd, v[2 * j + 1] * fwd);
  if (left > 0) {
    *reinterpret_cast<uint2*>(codes) = make_uint2(pc[0] | (pc[1] << 16), pc[2] | (pc[3] << 16));
    if (deq != nullptr) {
      uint32_t d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = decode_fp8x2<false>(pc[j]);
        d[j] = pack_bf16(f.x * inv, f.y * inv);
      }
      *reinterpret_cast<uint4*>(deq) = make_uint4(d[0], d[1], d[2], d[3]);
    }
  }
  return e;
}

// the exponents of `rows` rows from row0 and of the blocks [kb0, kb0 + blocks), staged as s_e[block][row], to their
// planes and the packed chunks: runs of the row index, words of four blocks
__device__ __forceinline__ void flush_exponents(const int8_t* s_e, const RowParams& p, int64_t row0, int rows, int pitch,
                                                int kb0, int blocks) {
  const int num_kb = p.width / p.block;
  const int tid = threadIdx.y * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y;
  blocks = min(blocks, num_kb - kb0);
  int8_t* plane = reinterpret_cast<int8_t*>(p.scale);
  // 2^k threads a block of columns, so that runs of rows go to neighbouring threads
  const int run = rows > 16 ? 32 : rows > 8 ? 16 : rows > 4 ? 8 : rows > 2 ? 4 : rows;
  for (int r = tid % run; r < rows; r += run)
    for (int kb = tid / run; kb < blocks; kb += threads / run)
      plane[(int64_t)(kb0 + kb) * p.rows + row0 + r] = s_e[kb * pitch + r];
  if (p.sf == nullptr) return;
  // kb0 is a multiple of four
  const int64_t k_groups = (num_kb + 3) >> 2;
  const int groups = (blocks + 3) >> 2;
  for (int r = tid % run; r < rows; r += run)
    for (int g = tid / run; g < groups; g += threads / run) {
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int kb = 4 * g + j;
        word |= (uint32_t)(kb < blocks ? e8m0_from_exp(s_e[kb * pitch + r]) : (uint8_t)127) << (8 * j);   // filled up with 2^0
      }
      *reinterpret_cast<uint32_t*>(p.sf + sf_chunk_offset(row0 + r, kb0 + 4 * g, k_groups)) = word;
    }
}

// blockDim = (threads of a row, rows side by side).  A thread holds 8 * NC values of its row in registers, and while it
// works on them the inputs of its next row are on their way (NC 1 and 2; bringing a wider row's next one to shared memory
// with cp.async measured slower: gate 16384 x 11008 to int8 210 -> 233 us, norm to block codes 308 -> 359 us).  The block
// walks `turns` rows for each of its blockDim.y places.  gridDim.y > 1 (only where no statistic spans the row) splits the
// row's columns.  NC = 0 walks a row of any width and loads it again for each pass.
template <int OP, bool BF16, bool VEC, bool BLOCK, int NC, int THREADS>
__global__ void __launch_bounds__(THREADS, !VEC && OP == OP_NORM ? 1 : THREADS == 256 ? 6 : THREADS == 384 ? 3 : THREADS == 512 ? 2 : 1)
row_quant_kernel(const RowParams p, const int turns) {
  __shared__ __align__(16) Slots s_sum, s_max;
  extern __shared__ int8_t s_e[];
  using E = Elem<BF16>;
  constexpr int kHeld = NC ? NC : 1;
  constexpr bool AHEAD = NC == 1 || NC == 2;
  let_next_start();
  wait_for_stream();
  const int step = blockDim.x, span = 8 * step, side = blockDim.y;
  const int col0 = kHeld * span * (int)blockIdx.y;
  const int first = (VEC ? 8 : 1) * (int)threadIdx.x + col0;
  const int chunks = NC ? NC : (p.width + span - 1) / span;
  const int block_rows = turns * side;
  const int64_t row0 = (int64_t)blockIdx.x * block_rows;
  const int64_t below = p.rows - row0;
  const int places = below < block_rows ? (int)below : block_rows;
  const E* a = reinterpret_cast<const E*>(p.a) + row0 * p.lda + first;
  const E* b = OP == OP_COPY || p.b == nullptr ? nullptr : reinterpret_cast<const E*>(p.b) + row0 * p.ldb + first;

  float v[kHeld][8];
  Inputs<OP, BF16, VEC> in[kHeld];
  // a place behind the last row loads that row once more and stores nothing
  auto load_row = [&](int place) {
    place = min(place, places - 1);
#pragma unroll
    for (int c = 0; c < kHeld; ++c)
      in[c].load(a + place * p.lda + c * span, b != nullptr ? b + place * p.ldb + c * span : nullptr, p.width - first - c * span, step);
  };
  if constexpr (AHEAD) load_row(threadIdx.y);
  if (step > 32) {      // absent warps' slots; ordered before the first read by the barrier in row_reduce
    const int tid = threadIdx.y * step + threadIdx.x;
    if (tid < 64 && (tid & 7) >= (step >> 5)) s_sum.v[0][tid] = s_sum.v[1][tid] = s_max.v[0][tid] = s_max.v[1][tid] = 0.f;
  }

  for (int turn = 0; turn * side < places; ++turn) {
    const int place = turn * side + (int)threadIdx.y;
    const bool live = place < places;
    const int64_t row = row0 + place;
    if constexpr (NC != 0) {
      if constexpr (!AHEAD) load_row(place);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if constexpr (OP == OP_NORM) {
          if (b != nullptr) in[c].add();
          if (live && p.h != nullptr)
            in[c].a.store(reinterpret_cast<E*>(p.h) + row * p.width + first + c * span, p.width - first - c * span, step);
        }
        in[c].value(v[c]);
      }
      if constexpr (AHEAD)
        if (turn + 1 < turns) load_row(place + side);
    }
    auto again = [&](int c) {      // NC = 0: chunk c once more
      const int at = min(place, places - 1);
      in[0].load(a + at * p.lda + c * span, b != nullptr ? b + at * p.ldb + c * span : nullptr, p.width - first - c * span, step);
      in[0].value(v[0]);
    };
    if constexpr (OP == OP_NORM) {
      static_assert(NC != 0, "the norm's row stays in registers");
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(v[c][j], v[c][j], sum);
      sum = row_reduce<false>(sum, s_sum.v[turn & 1]);
      const float rstd = rsqrtf(fmaf(sum, p.inv_width, p.eps));
      if (live && p.rstd != nullptr && threadIdx.x == 0) p.rstd[row] = rstd;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float w[8];
        if (p.w_bf16) load8<true, VEC>(w, p.w, first + c * span, p.width - first - c * span, step);
        else load8<false, VEC>(w, p.w, first + c * span, p.width - first - c * span, step);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] = v[c][j] * rstd * w[j];
      }
    }
    uint8_t* codes = p.codes + row * p.ldc + first;
    __nv_bfloat16* deq = p.deq != nullptr ? p.deq + row * p.width + first : nullptr;
    if constexpr (BLOCK) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int i0 = first - col0 + c * span;
        const int e = store_block(v[c], codes + c * span, deq != nullptr ? deq + c * span : nullptr,
                                  live ? p.width - first - c * span : 0, p.block);
        if (live && (i0 & (p.block - 1)) == 0) s_e[(i0 >> p.block_shift) * block_rows + place] = (int8_t)e;
      }
    } else {
      float am = 0.f;
#pragma unroll
      for (int c = 0; c < chunks; ++c) {
        if constexpr (NC == 0) again(c);
#pragma unroll
        for (int j = 0; j < 8; ++j) am = max_nan(am, fabsf(v[NC ? c : 0][j]));
      }
      am = row_reduce<true>(am, s_max.v[turn & 1]);
      const float s = row_scale(am);
      const float inv_s = __frcp_rn(s);
      if (live && threadIdx.x == 0) reinterpret_cast<float*>(p.scale)[row] = s;
#pragma unroll
      for (int c = 0; c < chunks; ++c) {
        if constexpr (NC == 0) again(c);
        if (live)
          store_int8<VEC>(v[NC ? c : 0], codes + c * span, deq != nullptr ? deq + c * span : nullptr, p.width - first - c * span,
                          step, s, inv_s);
      }
    }
  }
  if constexpr (BLOCK) {
    __syncthreads();
    flush_exponents(s_e, p, row0, places, block_rows, col0 >> p.block_shift, kHeld * span >> p.block_shift);
  }
}

// The same for many bf16 rows in int8 (OP_NORM or OP_COPY): one row for each place of a block, 8 * CH values a thread that
// wait in registers as they came, 2 bytes a value, and are formed again for each of the passes (sum of squares, maximum,
// codes).  Twice the values a thread halves what a row costs each of them (two reductions, the scale), and many small blocks
// hide one another's barriers.  32768 x 4096 with a residual 141 us (6.65 TB/s), the codes alone 64 us (6.3 TB/s); when both still
// divided near ties, 163 and 89 us here against 178 and 96 us in row_quant_kernel.
template <int OP, int CH>
__global__ void __launch_bounds__(256, 3) row_int8_kernel(const RowParams p) {
  __shared__ __align__(16) float s_sum[8], s_max[8];
  let_next_start();
  wait_for_stream();
  const int step = blockDim.x, span = 8 * step;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= p.rows) return;      // a whole warp: more than a warp a row has the block to itself
  if (step > 32 && threadIdx.x < 8 && (int)threadIdx.x >= (step >> 5)) s_sum[threadIdx.x] = s_max[threadIdx.x] = 0.f;
  const int first = 8 * (int)threadIdx.x;
  using R = Raw<true, true>;
  const __nv_bfloat16* a = reinterpret_cast<const __nv_bfloat16*>(p.a) + row * p.lda + first;
  R x[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) x[c].load(a + span * c, p.width - first - span * c, 0);
  float rstd = 1.f;
  if constexpr (OP == OP_NORM) {
    if (p.b != nullptr) {
      const __nv_bfloat16* b = reinterpret_cast<const __nv_bfloat16*>(p.b) + row * p.ldb + first;
      Inputs<OP, true, true> in;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        in.a = x[c];
        in.b.load(b + span * c, p.width - first - span * c, 0);
        in.add();
        x[c] = in.a;
      }
    }
    if (p.h != nullptr) {
      __nv_bfloat16* h = reinterpret_cast<__nv_bfloat16*>(p.h) + row * p.width + first;
#pragma unroll
      for (int c = 0; c < CH; ++c) x[c].store(h + span * c, p.width - first - span * c, 0);
    }
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(x[c].get(j), x[c].get(j), sum);
    rstd = rsqrtf(fmaf(row_reduce<false>(sum, s_sum), p.inv_width, p.eps));
    if (p.rstd != nullptr && threadIdx.x == 0) p.rstd[row] = rstd;
  }
  auto value = [&](float (&v)[8], int c) {
    if constexpr (OP == OP_NORM) {
      if (p.w_bf16) load8<true, true>(v, p.w, first + span * c, p.width - first - span * c, 0);
      else load8<false, true>(v, p.w, first + span * c, p.width - first - span * c, 0);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = OP == OP_NORM ? x[c].get(j) * rstd * v[j] : x[c].get(j);
  };
  float am = 0.f, v[8];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    value(v, c);
#pragma unroll
    for (int j = 0; j < 8; ++j) am = max_nan(am, fabsf(v[j]));
  }
  const float s = row_scale(row_reduce<true>(am, s_max));
  const float inv_s = __frcp_rn(s);
  if (threadIdx.x == 0) reinterpret_cast<float*>(p.scale)[row] = s;
  uint8_t* codes = p.codes + row * p.ldc + first;
  __nv_bfloat16* deq = p.deq != nullptr ? p.deq + row * p.width + first : nullptr;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    value(v, c);
    store_int8<true>(v, codes + span * c, deq != nullptr ? deq + span * c : nullptr, p.width - first - span * c, 0, s, inv_s);
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
  float inv_width;
};

// dx = rstd * (g - hat * mean(g * hat)) + dh with g = dy * w, hat = h * rstd;  dw = sum over rows of dy * hat.
// Bound by memory: 6 bytes in and 2 out a bf16 value.  blockDim = (threads of a row, rows side by side); a block walks
// every gridDim.x-th group of rows, a thread owns the same 8 * CH columns of all its rows, keeps the weight and its part of dw
// in registers and has the next row on its way while it works on this one.  32768 x 4096 bf16, the column sums included: 170 us
// (6.3 TB/s) with 16 values a thread, 178 us with 8 (189 us where the power cap holds the clock down: more instructions a
// value), 249 us without the row ahead.
template <bool BF16, bool VEC, int CH, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_norm_backward_kernel(const NormBwdParams p) {
  __shared__ __align__(16) Slots slots;
  extern __shared__ float s_acc[];       // (rows side by side, 8 * CH, threads of a row)
  using E = Elem<BF16>;
  const int step = blockDim.x, span = 8 * step, side = blockDim.y;
  let_next_start();
  wait_for_stream();
  const int first = (VEC ? 8 : 1) * (int)threadIdx.x;
  const int tid = threadIdx.y * step + threadIdx.x;
  if (tid < 64) slots.v[0][tid] = slots.v[1][tid] = 0.f;
  __syncthreads();
  float w[CH][8], acc[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if (p.w_bf16) load8<true, VEC>(w[c], p.w, first + c * span, p.width - first - c * span, step);
    else load8<false, VEC>(w[c], p.w, first + c * span, p.width - first - c * span, step);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[c][j] = 0.f;
  }

  Raw<BF16, VEC> dy[CH], h[CH], dh[CH];
  float rstd;
  // a row behind the last one is taken as zeros: it adds nothing
  auto load = [&](int64_t row) {
    const bool there = row < p.rows;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = first + c * span, n = there ? p.width - at : 0;
      dy[c].load(reinterpret_cast<const E*>(p.dy) + row * p.ld_dy + at, n, step);
      h[c].load(reinterpret_cast<const E*>(p.h) + row * p.ld_h + at, n, step);
      dh[c].load(reinterpret_cast<const E*>(p.dh) + row * p.ld_dh + at, p.dh != nullptr ? n : 0, step);
    }
    rstd = there ? __ldg(p.rstd + row) : 0.f;
  };
  int turn = 0;
  const int64_t stride = (int64_t)gridDim.x * side;
  int64_t group = (int64_t)blockIdx.x * side;
  load(group + threadIdx.y);
  for (; group < p.rows; group += stride, turn ^= 1) {
    const int64_t row = group + threadIdx.y;
    float g[CH][8], hat[CH][8];
    Raw<BF16, VEC> d[CH];
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        hat[c][j] = h[c].get(j) * rstd;
        acc[c][j] = fmaf(dy[c].get(j), hat[c][j], acc[c][j]);
        g[c][j] = dy[c].get(j) * w[c][j];
        sum = fmaf(g[c][j], hat[c][j], sum);
      }
      d[c] = dh[c];
    }
    const float r = rstd;
    load(row + stride);
    const float mean = row_reduce<false>(sum, slots.v[turn]) * p.inv_width;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int j = 0; j < 8; ++j) g[c][j] = fmaf(r, g[c][j] - hat[c][j] * mean, d[c].get(j));
      const int at = first + c * span;
      if (row < p.rows) store8<BF16, VEC>(g[c], p.dx, row * (int64_t)p.width + at, p.width - at, step);
    }
  }
  if (side > 1) {
#pragma unroll
    for (int k = 0; k < 8 * CH; ++k) s_acc[(threadIdx.y * 8 * CH + k) * step + threadIdx.x] = acc[k / 8][k % 8];
    __syncthreads();
    if (threadIdx.y != 0) return;
    for (int y = 1; y < side; ++y)
#pragma unroll
      for (int k = 0; k < 8 * CH; ++k) acc[k / 8][k % 8] += s_acc[(y * 8 * CH + k) * step + threadIdx.x];
  }
#pragma unroll
  for (int c = 0; c < CH; ++c)
    store8<false, VEC>(acc[c], p.dw, (int64_t)blockIdx.x * p.width + first + c * span, p.width - first - c * span, step);
}

// The same for rows of more than 8192 values: a block's rows are read twice, the second time from L2, and its part of dw
// lies in shared memory.
template <bool BF16, bool VEC>
__global__ void __launch_bounds__(1024) rms_norm_backward_wide_kernel(const NormBwdParams p) {
  __shared__ __align__(16) Slots slots;
  extern __shared__ float s_acc[];       // (8 * chunks, threads)
  const int step = blockDim.x, span = 8 * step;
  const int first = (VEC ? 8 : 1) * (int)threadIdx.x;
  const int chunks = (p.width + span - 1) / span;
  let_next_start();
  wait_for_stream();
  for (int k = 0; k < 8 * chunks; ++k) s_acc[k * step + threadIdx.x] = 0.f;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const float rstd = __ldg(p.rstd + row);
    float g[8], hat[8], w[8], sum = 0.f;
    auto load = [&](int c) {
      const int i0 = first + c * span, left = p.width - i0;
      load8<BF16, VEC>(g, p.dy, row * p.ld_dy + i0, left, step);
      load8<BF16, VEC>(hat, p.h, row * p.ld_h + i0, left, step);
      if (p.w_bf16) load8<true, VEC>(w, p.w, i0, left, step);
      else load8<false, VEC>(w, p.w, i0, left, step);
    };
    for (int c = 0; c < chunks; ++c) {
      load(c);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(g[j] * w[j], hat[j] * rstd, sum);
    }
    const float mean = row_reduce<false>(sum, slots.v[turn]) * p.inv_width;
    for (int c = 0; c < chunks; ++c) {
      load(c);
      const int i0 = first + c * span, left = p.width - i0;
      float d[8];
      load8<BF16, VEC>(d, p.dh, row * p.ld_dh + i0, p.dh != nullptr ? left : 0, step);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        hat[j] *= rstd;
        s_acc[(8 * c + j) * step + threadIdx.x] += g[j] * hat[j];
        d[j] = fmaf(rstd, g[j] * w[j] - hat[j] * mean, d[j]);
      }
      store8<BF16, VEC>(d, p.dx, row * (int64_t)p.width + i0, left, step);
    }
  }
  for (int c = 0; c < chunks; ++c) {
    float a[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = s_acc[(8 * c + j) * step + threadIdx.x];
    store8<false, VEC>(a, p.dw, (int64_t)blockIdx.x * p.width + first + c * span, p.width - first - c * span, step);
  }
}

// out[c] = sum over r of partial[r, c]; 32 columns a block, the rows dealt to 16 warps and joined in a fixed order
__global__ void column_sum_kernel(const float* __restrict__ partial, int rows, int width, float* __restrict__ out) {
  __shared__ float s[16][32];
  let_next_start();
  wait_for_stream();
  const int c = blockIdx.x * 32 + threadIdx.x;
  float t = 0.f;
  if (c < width) {
#pragma unroll 8
    for (int r = threadIdx.y; r < rows; r += 16) t += partial[(int64_t)r * width + c];
  }
  s[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.y == 0 && c < width) {
#pragma unroll
    for (int k = 1; k < 16; ++k) t += s[k][threadIdx.x];
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

// sigma = 1/(1+e^-g): dgate = dy * u * sigma * (1 + g (1 - sigma)), dup = dy * g * sigma.  Bound by memory in either type:
// FP32 8192 x 11008 268 us with the longer sigma, 273 us with the short one; bf16 16384 x 11008 273 us.
template <bool BF16, bool VEC>
__global__ void silu_mul_backward_kernel(const GateBwdParams p) {
  let_next_start();
  wait_for_stream();
  const int step = blockDim.x;
  const int i0 = (VEC ? 8 : 1) * (int)threadIdx.x + 8 * step * (int)blockIdx.y;
  const int64_t row = blockIdx.x;
  float d[8], g[8], u[8];
  load8<BF16, VEC>(d, p.dy, row * p.ld_dy + i0, p.width - i0, step);
  load8<BF16, VEC>(g, p.gate, row * p.ld_gate + i0, p.width - i0, step);
  load8<BF16, VEC>(u, p.up, row * p.ld_up + i0, p.width - i0, step);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float sig = BF16 ? sigmoid(g[j]) : sigmoid_f32(g[j]);
    const float ds = d[j] * sig;
    const float dg = ds * u[j] * fmaf(g[j], 1.f - sig, 1.f);
    u[j] = ds * g[j];
    g[j] = dg;
  }
  store8<BF16, VEC>(g, p.dgate, row * p.ld_dgate + i0, p.width - i0, step);
  store8<BF16, VEC>(u, p.dup, row * p.ld_dup + i0, p.width - i0, step);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
bool aligned16(const void* ptr, int64_t ld, int elem) {
  return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0 && ((ld * elem) & 15) == 0;
}

int round32(int x) { return (x + 31) & ~31; }

int block_shift(int block) { return block == 128 ? 7 : block == 64 ? 6 : 5; }

// Threads and values a thread (8 * NC), by the row's width, and rows a block.  Measured at 32768 x 4096 bf16, block 64, with a
// residual: 256 threads x 16 values with the next row on its way 149 us (6.3 TB/s), without 172 us; 128 threads x 32 values
// 215 us; 8 rows a block 149 us, 16 rows 155 us, 1 row 230 us (nothing ahead, and the exponents leave as single bytes).
// Narrower rows want more of them: 16384 x 1024 27 us with 8 rows, 23 us with 32.  A row of more than 8192 values takes 32 a
// thread and no load ahead (registers); up to 12288 three blocks share an SM: gate 16384 x 11008 to int8 153 us (5.9 TB/s),
// two blocks 195 us.  That form keeps its values in 56 registers; the norm, FP32 and single-value forms spill 8 to 276 bytes a
// thread there (norm 16384 x 11008 to int8 299 us, 4.2 TB/s) and were not timed with two blocks.  The gated block form has no
// row statistic: 128 threads x 8 values walk 16 rows of 1024 columns, 16384 x 11008 155 us (5.8 TB/s), with bf16 values 208 us
// (6.1 TB/s); 256 threads 175 and 234 us (before the shorter sigmoid).
// Rows off 16-byte boundaries take single values and are bound by their instructions: 16384 x 1001 FP32 norm 49 us (3.7 TB/s).
template <int OP, bool BF16, bool VEC, bool BLOCK>
int launch_row(const RowParams& p, cudaStream_t stream) {
  constexpr bool kSplit = OP != OP_NORM && BLOCK;       // the row's columns over several blocks
  const int units = (p.width + 7) / 8;
  if constexpr (OP != OP_GATE && BF16 && VEC && !BLOCK) {
    // rows enough for every SM many times over; fewer are done sooner with more threads a row
    if (units > 32 && units <= 1024 && p.rows >= 16 * (int64_t)sm_count()) {
      const int threads = units <= 128 ? 32 : round32((units + 3) / 4), side = threads == 32 ? 4 : 1;
      const unsigned blocks = (unsigned)((p.rows + side - 1) / side);
      if (units <= 64) CUDA_TRY(launch_early(row_int8_kernel<OP, 2>, dim3(blocks), dim3(threads, side), 0, stream, p));
      else CUDA_TRY(launch_early(row_int8_kernel<OP, 4>, dim3(blocks), dim3(threads, side), 0, stream, p));
      return TCFP_OK;
    }
  }
  int nc, threads, col_blocks = 1;
  if (kSplit) {
    nc = 1;
    // even shares of up to 128 threads, in multiples of four scale blocks (a word of packed scale factors)
    const int grain = p.block == 128 ? 64 : 32;
    col_blocks = (units + 127) / 128;
    if (col_blocks > 65535) col_blocks = (units + 255) / 256;      // what gridDim.y can hold: the widest rows take 256 threads
    threads = ((units + col_blocks - 1) / col_blocks + grain - 1) / grain * grain;
  } else {
    nc = units <= 64 ? 1 : units <= 1024 ? 2 : units <= 4096 ? 4 : 0;
    threads = nc == 0 ? 1024 : units <= 16 ? 16 : round32((units + nc - 1) / nc);
  }
  int side = threads < 256 && !kSplit ? 256 / threads : 1;
  if (side > p.rows) side = threads == 16 ? (int)((p.rows + 1) & ~1) : (int)p.rows;      // whole warps
  // first enough blocks for every SM, twice over; then as many rows as are worth it
  const int64_t resident = (int64_t)sm_count() * 2 * ((nc == 1 ? 1536 : nc == 4 && threads <= 384 ? 1152 : 1024) / (threads * side));
  const int64_t fair = (p.rows * col_blocks + resident - 1) / resident;
  const int most = kSplit ? 16 : p.width >= 4096 ? 8 : p.width <= 1024 ? 32 : 32768 / p.width;
  const int block_rows = (int)(fair < most ? fair : most);
  const int turns = (block_rows + side - 1) / side;
  const dim3 grid((unsigned)((p.rows + turns * side - 1) / (turns * side)), (unsigned)col_blocks);
  const dim3 block((unsigned)threads, (unsigned)side);
  const size_t smem = BLOCK ? (size_t)nc * threads * 8 / p.block * turns * side : 0;
#define ROW(NC, THREADS) CUDA_TRY(launch_early(row_quant_kernel<OP, BF16, VEC, BLOCK, NC, THREADS>, grid, block, smem, stream, p, turns))
  if (nc == 1) ROW(1, 256);
  if constexpr (!kSplit) {
    if (nc == 2) ROW(2, 512);
    if (nc == 4 && threads <= 384) ROW(4, 384);
    if (nc == 4 && threads > 384) ROW(4, 1024);
    if constexpr (OP != OP_NORM)
      if (nc == 0) ROW(0, 1024);
  }
#undef ROW
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

constexpr int kNormBwdWidth = 8192;      // 8 values for each of 1024 threads

// threads of a row, rows side by side and blocks of the norm's backward pass: one set of resident blocks
struct NormBwdShape {
  int chunks, threads, side, blocks;
};
NormBwdShape norm_bwd_shape(int64_t rows, int64_t width, bool two) {
  const int units = (int)((width + 7) / 8);
  NormBwdShape s;
  s.chunks = two && units > 32 && units <= 1024 ? 2 : 1;
  // blocks of up to 512 threads have 128 registers a thread: FP32 rows and narrow loads spill with 64
  s.threads = units > 1024 ? 1024 : units <= 16 ? 16 : round32((units + s.chunks - 1) / s.chunks);
  s.side = s.threads < 256 ? 256 / s.threads : 1;
  const int64_t groups = (rows + s.side - 1) / s.side;
  const int64_t resident = (int64_t)sm_count() * (width > kNormBwdWidth ? 1 : s.threads > 512 ? 1 : 512 / (s.threads * s.side));
  s.blocks = (int)(groups < resident ? groups : resident);
  return s;
}

template <bool BF16, bool VEC>
int launch_norm_bwd(const NormBwdParams& p, const NormBwdShape& s, cudaStream_t stream) {
  if (p.width <= kNormBwdWidth) {
    const size_t smem = s.side > 1 ? (size_t)s.side * s.threads * 8 * s.chunks * sizeof(float) : 0;
    if constexpr (BF16 && VEC) {
      if (s.chunks == 2) {
        CUDA_TRY(launch_early(rms_norm_backward_kernel<BF16, VEC, 2, 512>, dim3(s.blocks), dim3(s.threads, s.side), smem, stream, p));
        return TCFP_OK;
      }
    }
    if (s.threads <= 512) CUDA_TRY(launch_early(rms_norm_backward_kernel<BF16, VEC, 1, 512>, dim3(s.blocks), dim3(s.threads, s.side), smem, stream, p));
    else CUDA_TRY(launch_early(rms_norm_backward_kernel<BF16, VEC, 1, 1024>, dim3(s.blocks), dim3(s.threads, s.side), smem, stream, p));
  } else {
    const int smem = (p.width + 8191) / 8192 * 8192 * (int)sizeof(float);
    static bool done[64] = {false};
    int dev = 0;
    CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return fail(TCFP_ERR_UNSUPPORTED, "device index %d out of range", dev);
    if (!done[dev]) {
      CUDA_TRY(cudaFuncSetAttribute(rms_norm_backward_wide_kernel<BF16, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    kMaxNormWidth * (int)sizeof(float)));
      done[dev] = true;
    }
    CUDA_TRY(launch_early(rms_norm_backward_wide_kernel<BF16, VEC>, dim3(s.blocks), dim3(s.threads), smem, stream, p));
  }
  return TCFP_OK;
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
              sf_out, reinterpret_cast<__nv_bfloat16*>(deq_bf16_out), rows, (int)width, block_size, block_shift(block_size), 1.f / (float)width};
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
              reinterpret_cast<__nv_bfloat16*>(deq_bf16_out), rows, (int)width, block_size, block_shift(block_size), 1.f / (float)width};
  const int rc = check_row("tcfp_silu_mul_quantize", p, dtype, dtype == TCFP_BF16 ? 2 : 4);
  if (rc != TCFP_OK) return rc;
  return dtype == TCFP_BF16 ? dispatch_row<OP_GATE, true>(p, (cudaStream_t)stream) : dispatch_row<OP_GATE, false>(p, (cudaStream_t)stream);
}

extern "C" int32_t tcfp_int8_quantize_rows(const void* x, int64_t ld_x, int32_t dtype, uint8_t* codes, int64_t ld_codes,
                                           float* scale_out, void* deq_bf16_out, int64_t rows, int64_t width, void* stream) {
  if (width > kMaxGateWidth) return fail(TCFP_ERR_UNSUPPORTED, "tcfp_int8_quantize_rows: width %lld", (long long)width);
  RowParams p{x, nullptr, ld_x, 0, nullptr, 0, 0.f, nullptr, nullptr, codes, ld_codes, scale_out, nullptr,
              reinterpret_cast<__nv_bfloat16*>(deq_bf16_out), rows, (int)width, 0, block_shift(0), 1.f / (float)width};
  const int rc = check_row("tcfp_int8_quantize_rows", p, dtype, dtype == TCFP_BF16 ? 2 : 4);
  if (rc != TCFP_OK) return rc;
  return dtype == TCFP_BF16 ? dispatch_row<OP_COPY, true>(p, (cudaStream_t)stream) : dispatch_row<OP_COPY, false>(p, (cudaStream_t)stream);
}

extern "C" size_t tcfp_rms_norm_backward_workspace_bytes(int64_t rows, int64_t width) {
  if (rows < 1 || width < 1 || width > kMaxNormWidth) return 0;
  // the call's alignment, which it does not know, decides between the two shapes
  const int one = norm_bwd_shape(rows, width, false).blocks, two = norm_bwd_shape(rows, width, true).blocks;
  return (size_t)(one > two ? one : two) * (size_t)width * sizeof(float);
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
  bool vec = width % 8 == 0 && aligned16(dy, ld_dy, e) && aligned16(h, ld_h, e) && (!dh || aligned16(dh, ld_dh, e)) &&
             aligned16(weight, 0, 1) && aligned16(dx, 0, 1) && aligned16(dw, 0, 1) && aligned16(workspace, 0, 1);
  const NormBwdShape shape = norm_bwd_shape(rows, width, vec && dtype == TCFP_BF16);
  const int blocks = shape.blocks;
  const NormBwdParams p{dy, h, dh, ld_dy, ld_h, ld_dh, rstd, weight, w_dtype == TCFP_BF16, dx,
                        blocks == 1 ? dw : reinterpret_cast<float*>(workspace), rows, (int)width, 1.f / (float)width};
  int rc;
  if (dtype == TCFP_BF16) rc = vec ? launch_norm_bwd<true, true>(p, shape, stream) : launch_norm_bwd<true, false>(p, shape, stream);
  else rc = vec ? launch_norm_bwd<false, true>(p, shape, stream) : launch_norm_bwd<false, false>(p, shape, stream);
  if (rc != TCFP_OK || blocks == 1) return rc;
  CUDA_TRY(launch_early(column_sum_kernel, dim3((unsigned)((width + 31) / 32)), dim3(32, 16), 0, stream, p.dw, blocks, (int)width, dw));
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
    if (vec) CUDA_TRY(launch_early(silu_mul_backward_kernel<true, true>, grid, dim3(threads), 0, stream, p));
    else CUDA_TRY(launch_early(silu_mul_backward_kernel<true, false>, grid, dim3(threads), 0, stream, p));
  } else {
    if (vec) CUDA_TRY(launch_early(silu_mul_backward_kernel<false, true>, grid, dim3(threads), 0, stream, p));
    else CUDA_TRY(launch_early(silu_mul_backward_kernel<false, false>, grid, dim3(threads), 0, stream, p));
  }
  return TCFP_OK;
}
