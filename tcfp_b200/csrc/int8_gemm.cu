// int8 product with a scale for each token and each channel (sm_100a).
//
//   out[m,n] = (sum_k a[m,k] b[n,k]) * s_a[m] * s_b[n] + bias[n]
//
// The sum is an exact 32-bit integer; the two scales are constant along k, so they are applied once, to the finished
// sum.  Two kernels on tcgen05.mma kind::i8, both fed by TMA through a ring of 128-byte-wide stages of K:
//
//   int8_pair_kernel  prompts: a pair of CTAs (cta_group::2) owns a 256 x 256 output tile, as the FP8 pair kernel does.
//                     Bound by the tensor pipe: 8192 x 12288 x 4096 252 us, 3.27 Pop/s (98 % of twice the measured bf16
//                     rate).  The channel scales of a tile wait in shared memory: with every thread reading them from
//                     global memory the epilogue took 7 us a tile and set the pace for K below 2048.
//   int8_few_kernel   few tokens: bound by the weight's bytes, so the weight takes the 128 rows of the MMA and the tokens
//                     its 16..128 columns, and the CTAs of a cluster split K; the partial sums meet through distributed
//                     shared memory.  Integer sums do not depend on the split.  22016 x 4096: 19 us for 1 to 32 tokens
//                     (4.7 TB/s), 12288 x 4096 12 us (4.2 TB/s).
//
// Every wait is bounded; see sm100_ptx.cuh.
#include <cuda.h>

#include "common.cuh"
#include "launch.h"
#include "sm100_ptx.cuh"

namespace tcfp {
namespace {

constexpr int kThreads = 192;       // warp 0 TMA, warp 1 MMA and TMEM, warps 2-5 epilogue
constexpr int kStageK = 128;        // bytes of K in a stage: one swizzle row
constexpr int kMmaK = 32;
constexpr int kTile = 16384;        // 128 rows x 128 bytes

struct Int8Params {
  const float *s_a, *s_b, *bias;
  void* out;
  int M, N, K;
  int k_stages;
  int group_m;
  int out_bf16;
  int stages;        // of the ring (few tokens)
  int wide_out;      // rows of out start on boundaries of four elements
  unsigned int* status;
};

// instruction descriptor of kind::i8: S32 accumulator, both operands signed and K-major
__device__ __forceinline__ uint32_t i8_idesc(uint32_t m, uint32_t n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
template <int CTAS>
__device__ __forceinline__ void tc_mma_i8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  if constexpr (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum)
        : "memory");
}

// whether all 128 threads that share barrier `id` got through a wait: they go on or leave together, so that none is missing
// at a barrier
__device__ __forceinline__ bool epi_all(bool ok, int id = 1) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "bar.red.and.pred p, %2, 128, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(all)
      : "r"((uint32_t)ok), "r"(id)
      : "memory");
  return all != 0;
}
__device__ __forceinline__ void epi_sync(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }

__device__ __forceinline__ float scaled(int acc, float s_a, float s_b, float bias) {
  return fmaf(__int2float_rn(acc) * s_a, s_b, bias);
}

// ---------------------------------------------------------------------------
// prompts: CTA pairs, 256 x 256 tiles
// ---------------------------------------------------------------------------
constexpr int kPairStages = 5;
constexpr int kPairStageBytes = 2 * kTile;
constexpr int kPieceBytes = 16384;            // 128 rows x 128 bytes of staged output
constexpr int kColumnBytes = 2 * 2 * 256 * 4;   // channel scales and bias of two tiles
constexpr int kPairSmem = 1024 + kPairStages * kPairStageBytes + 2 * kPieceBytes + kColumnBytes + 256;

// G groups of four epilogue warps share a tile's columns
template <bool OUT_BF16, int G>
__global__ void __launch_bounds__(64 + 128 * G, 1)
int8_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                 const __grid_constant__ CUtensorMap tm_out, const Int8Params p, const int tma_store) {
  constexpr int kStages = kPairStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* staging = smem + kStages * kPairStageBytes;
  float* columns = reinterpret_cast<float*>(staging + 2 * kPieceBytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + 2 * kPieceBytes + kColumnBytes);
  const uint32_t bar_full = smem_u32(bars), bar_empty = smem_u32(bars + kStages);
  const uint32_t bar_tfull = smem_u32(bars + 2 * kStages), bar_tempty = smem_u32(bars + 2 * kStages + 2);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int tiles_m = (p.M + 255) / 256, tiles_n = (p.N + 255) / 256;
  const int num_tiles = tiles_m * tiles_n;
  // tiles in groups of group_m rows, down the rows first, so that a wave of pairs shares few columns of b
  auto coords = [&](int tile, int& mb, int& nb) {
    const int per_group = p.group_m * tiles_n;
    const int first = tile / per_group * p.group_m;
    const int gm = min(tiles_m - first, p.group_m);
    const int in_group = tile % per_group;
    mb = first + in_group % gm;
    nb = in_group / gm;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_tfull + 8 * b, 1);
      mbar_init(bar_tempty + 8 * b, 8 * G);  // one arrival per epilogue warp of both CTAs
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_a);
    prefetch_tmap(&tm_b);
    if (tma_store) prefetch_tmap(&tm_out);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_holder), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // both CTAs' barriers exist before anything remote touches them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  let_next_start();
  wait_for_stream();

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool live = true;
      for (int tile = pair; live && tile < num_tiles; tile += num_pairs) {
        int mb, nb;
        coords(tile, mb, nb);
        const int row_a = mb * 256 + (int)rank * 128, row_b = nb * 256 + (int)rank * 128;
        for (int ks = 0; ks < p.k_stages; ++ks) {
          if (!mbar_wait(bar_empty + 8 * stage, phase ^ 1, abort_flag, p.status)) { live = false; break; }
          const uint32_t full_leader = mapa(bar_full + 8 * stage, 0);
          if (rank == 0) mbar_expect_tx(bar_full + 8 * stage, 2 * kPairStageBytes);
          const uint32_t sa = smem_u32(smem + stage * kPairStageBytes);
          tma_load_2d_pair(sa, &tm_a, ks * kStageK, row_a, full_leader);
          tma_load_2d_pair(sa + kTile, &tm_b, ks * kStageK, row_b, full_leader);
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = i8_idesc(256, 256);
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      bool live = true;
      for (int tile = pair; live && tile < num_tiles; tile += num_pairs) {
        if (!mbar_wait(bar_tempty + 8 * buf, buf_phase ^ 1, abort_flag, p.status)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(buf * 256);
        for (int ks = 0; ks < p.k_stages; ++ks) {
          if (!mbar_wait(bar_full + 8 * stage, phase, abort_flag, p.status)) { live = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * kPairStageBytes);
#pragma unroll
          for (int j = 0; j < kStageK / kMmaK; ++j)
            tc_mma_i8<2>(d_tmem, make_desc(sa + j * kMmaK, 16, 1024, 2), make_desc(sa + kTile + j * kMmaK, 16, 1024, 2), idesc,
                         (ks | j) != 0 ? 1u : 0u);
          tc_commit_pair(bar_empty + 8 * stage);
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
        if (!live) break;
        tc_commit_pair(bar_tfull + 8 * buf);
        if (++buf == 2) { buf = 0; buf_phase ^= 1; }
      }
    }
    __syncwarp();
  } else {
    // epilogue: both CTAs, 128 rows each; a group takes its columns 32 at a time and has the next ones on their way.  One group
    // alternates between the two staging pieces, two have one each
    constexpr int kCols = 256 / G;
    constexpr int kPieceCols = OUT_BF16 ? 64 : 32;       // columns in a 128-byte row of the staging piece
    constexpr int kElem = OUT_BF16 ? 2 : 4;
    const int group = G == 2 && warp >= 6, id = 1 + group;
    const int q = warp & 3;
    const int r_local = q * 32 + lane;
    const bool issuer = threadIdx.x == 64 + 128 * group;
    uint8_t* piece = staging + group * kPieceBytes;
    int buf = 0;
    uint32_t buf_phase = 0;
    for (int tile = pair; tile < num_tiles; tile += num_pairs) {
      int mb, nb;
      coords(tile, mb, nb);
      const int row0 = mb * 256 + (int)rank * 128, col0 = nb * 256 + group * kCols;
      const float s_a = row0 + r_local < p.M ? __ldg(p.s_a + row0 + r_local) : 0.f;
      // these columns' scales and bias; those of the tile before may still be read from the other buffer
      float* s_col = columns + (buf * G + group) * 2 * kCols;
      for (int c = (threadIdx.x - 64) & 127; c < kCols; c += 128) {
        const int n = col0 + c;
        s_col[c] = n < p.N ? __ldg(p.s_b + n) : 0.f;
        s_col[kCols + c] = n < p.N && p.bias ? __ldg(p.bias + n) : 0.f;
      }
      if (!epi_all(mbar_wait(bar_tfull + 8 * buf, buf_phase, abort_flag, p.status), id)) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * 256 + group * kCols);
      uint32_t v[32];
      tmem_ld32(t_row, v);
#pragma unroll 1
      for (int g = 0; g < kCols / 32; ++g) {
        tmem_ld_wait();
        float o[32];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float4 sb = reinterpret_cast<const float4*>(s_col + g * 32)[c];
          const float4 bi = reinterpret_cast<const float4*>(s_col + kCols + g * 32)[c];
          o[4 * c] = scaled((int)v[4 * c], s_a, sb.x, bi.x);
          o[4 * c + 1] = scaled((int)v[4 * c + 1], s_a, sb.y, bi.y);
          o[4 * c + 2] = scaled((int)v[4 * c + 2], s_a, sb.z, bi.z);
          o[4 * c + 3] = scaled((int)v[4 * c + 3], s_a, sb.w, bi.w);
        }
        if (g < kCols / 32 - 1) {
          tmem_ld32(t_row + (g + 1) * 32, v);       // on its way while this piece is written
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa(bar_tempty + 8 * buf, 0));
        }
        // a piece may be rewritten once the store that last used it has read it: with one group that is the piece before last,
        // with two groups the last one
        if (!OUT_BF16 || (g & 1) == 0) {
          if (issuer) {
            if constexpr (G == 1) bulk_wait_read1();
            else bulk_wait_read0();
          }
          epi_sync(id);
        }
        uint8_t* line = piece + r_local * 128;
        if constexpr (!OUT_BF16) {
#pragma unroll
          for (int c = 0; c < 8; ++c)
            *reinterpret_cast<float4*>(line + ((c ^ (r_local & 7)) << 4)) =
                make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              __nv_bfloat162 b = __floats2bfloat162_rn(o[8 * c + 2 * k], o[8 * c + 2 * k + 1]);
              w[k] = *reinterpret_cast<uint32_t*>(&b);
            }
            *reinterpret_cast<uint4*>(line + ((((g & 1) * 4 + c) ^ (r_local & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        if (OUT_BF16 && (g & 1) == 0) continue;
        const int nst = col0 + (OUT_BF16 ? (g >> 1) : g) * kPieceCols;
        if (tma_store) {
          fence_async_smem();
          epi_sync(id);
          if (issuer) {
            // a piece outside the output commits an empty group, so that the wait above counts pieces
            if (nst < p.N && row0 < p.M) tma_store_2d(&tm_out, smem_u32(piece), nst, row0);
            bulk_commit();
          }
        } else {
          // rows of out that do not start on 16-byte boundaries: a warp writes a row's piece, neighbouring lanes neighbouring
          // columns
          epi_sync(id);
          const int rows = min(128, p.M - row0), cols = min(kPieceCols, p.N - nst);
#pragma unroll 4
          for (int r = q; r < rows; r += 4)
#pragma unroll
            for (int c = lane; c < kPieceCols; c += 32)
              if (c < cols) {
                const uint8_t* src = piece + r * 128 + (((c * kElem >> 4) ^ (r & 7)) << 4) + (c * kElem & 15);
                const int64_t at = (int64_t)(row0 + r) * p.N + nst + c;
                if constexpr (OUT_BF16) reinterpret_cast<uint16_t*>(p.out)[at] = *reinterpret_cast<const uint16_t*>(src);
                else reinterpret_cast<uint32_t*>(p.out)[at] = *reinterpret_cast<const uint32_t*>(src);
              }
        }
        if constexpr (G == 1) piece = staging + (piece == staging ? kPieceBytes : 0);
      }
      if (++buf == 2) { buf = 0; buf_phase ^= 1; }
    }
    if (issuer) bulk_wait0();
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    for (int i = 0; i < 20; ++i) __nanosleep(1000);
  }
  cluster_sync_all();   // the peer may still be reading operands / signalling barriers of this CTA
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---------------------------------------------------------------------------
// few tokens: the weight on the rows of the MMA, K split over the CTAs of a cluster
// ---------------------------------------------------------------------------
template <int NT>
struct Few {
  static constexpr int kStageBytes = kTile + NT * kStageK;
  static constexpr int kPartBytes = NT * 128 * 4;           // the partial sums reuse the stages
  static constexpr int kMinStages = (kPartBytes + kStageBytes - 1) / kStageBytes > 2 ? (kPartBytes + kStageBytes - 1) / kStageBytes : 2;
  static constexpr uint32_t kTmemCols = NT < 32 ? 32 : NT;
  static constexpr int smem(int stages) { return 1024 + stages * kStageBytes + 256; }
};
constexpr int kMaxFewStages = 12;                            // of the barriers behind the stages

// volatile keeps it behind the cluster barrier
__device__ __forceinline__ int4 ld_cluster_v4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

// gridDim = (S, weight tiles, token tiles), cluster = (S, 1, 1)
template <int NT, int S>
__global__ void __launch_bounds__(kThreads)
int8_few_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Int8Params p) {
  using F = Few<NT>;
  const int kStages = p.stages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStages * F::kStageBytes);
  const uint32_t bar_full = smem_u32(bars), bar_empty = smem_u32(bars + kStages), bar_done = smem_u32(bars + 2 * kStages);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x;
  const int n0 = blockIdx.y * 128, t0 = blockIdx.z * NT;
  const int ks0 = p.k_stages * rank / S, ks1 = p.k_stages * (rank + 1) / S;

  // warp 0: one thread feeds the ring; the first round of loads does not wait for the rest of the block
  int ks = ks0, stage = 0;
  uint32_t phase = 0;
  auto load = [&]() {
    mbar_expect_tx(bar_full + 8 * stage, F::kStageBytes);
    const uint32_t sw = smem_u32(smem + stage * F::kStageBytes);
    tma_load_2d(sw, &tm_w, ks * kStageK, n0, bar_full + 8 * stage);
    tma_load_2d(sw + kTile, &tm_x, ks * kStageK, t0, bar_full + 8 * stage);
    if (++stage == kStages) { stage = 0; phase ^= 1; }
    ++ks;
  };
  const bool feeder = warp == 0 && elect_one();
  let_next_start();
  if (feeder) {
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_x);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
    wait_for_stream();
    while (ks < ks1 && ks - ks0 < kStages) load();
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_holder), F::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  wait_for_stream();      // every role, so that no bounded wait below counts the time of the kernel before this one
  const uint32_t tmem_base = *tmem_holder;

  if (warp == 0) {
    if (feeder) {
      while (ks < ks1 && mbar_wait(bar_empty + 8 * stage, phase ^ 1, abort_flag, p.status)) load();
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = i8_idesc(128, NT);
      int stage = 0;
      uint32_t phase = 0;
      bool live = true;
      for (int ks = ks0; ks < ks1; ++ks) {
        if (!mbar_wait(bar_full + 8 * stage, phase, abort_flag, p.status)) { live = false; break; }
        tc_fence_after();
        const uint32_t sw = smem_u32(smem + stage * F::kStageBytes);
#pragma unroll
        for (int j = 0; j < kStageK / kMmaK; ++j)
          tc_mma_i8<1>(tmem_base, make_desc(sw + j * kMmaK, 16, 1024, 2), make_desc(sw + kTile + j * kMmaK, 16, 1024, 2), idesc,
                       (ks != ks0 || j != 0) ? 1u : 0u);
        tc_commit(bar_empty + 8 * stage);
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
      if (live) tc_commit(bar_done);
    }
    __syncwarp();
  }
  // The sums go to shared memory as (token, weight row) and meet there: the CTAs of the cluster take the tokens in turn, a
  // warp a token, a lane four neighbouring channels.
  const int tokens = min(NT, p.M - t0);
  int* part = reinterpret_cast<int*>(smem);       // every load and MMA is done by then
  bool live = true;
  const int n = n0 + lane * 4;
  float s_b[4], bias[4];
  if (warp >= 2) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s_b[k] = n + k < p.N ? __ldg(p.s_b + n + k) : 0.f;
      bias[k] = n + k < p.N && p.bias ? __ldg(p.bias + n + k) : 0.f;
    }
    live = epi_all(mbar_wait(bar_done, 0, abort_flag, p.status));
    if (live) {
      tc_fence_after();
      const int row = ((warp & 3) << 5) | lane;   // warps 2-5 cover the four lane quarters of TMEM
      for (int c = 0; c < tokens; c += 32) {
        uint32_t v[32];
        tmem_ld32(tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < (NT < 32 ? NT : 32); ++i) part[(c + i) * 128 + row] = (int)v[i];
      }
      tc_fence_before();
    }
  }
  __syncwarp();
  if constexpr (S > 1) cluster_sync_all();
  else if (warp >= 2) epi_bar_sync();
  if (warp >= 2 && live) {
    constexpr int kBatch = S >= 8 ? 2 : 16 / S > 8 ? 8 : 16 / S;     // tokens whose sums are on their way at once
    const uint32_t mine = smem_u32(part) + lane * 16;
    for (int t = rank + S * (warp - 2); t < tokens; t += 4 * S * kBatch) {
      int4 v[kBatch][S];
      float s_a[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int at = min(t + 4 * S * b, tokens - 1);
        s_a[b] = __ldg(p.s_a + t0 + at);
#pragma unroll
        for (int r = 0; r < S; ++r) v[b][r] = ld_cluster_v4(S > 1 ? mapa(mine + at * 512, r) : mine + at * 512);
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int at = t + 4 * S * b;
        if (at >= tokens) break;
        int acc[4] = {v[b][0].x, v[b][0].y, v[b][0].z, v[b][0].w};
#pragma unroll
        for (int r = 1; r < S; ++r) {
          acc[0] += v[b][r].x; acc[1] += v[b][r].y; acc[2] += v[b][r].z; acc[3] += v[b][r].w;
        }
        float o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = scaled(acc[k], s_a[b], s_b[k], bias[k]);
        const int64_t where = (int64_t)(t0 + at) * p.N + n;
        if (p.wide_out) {          // N is a multiple of 4: four channels or none
          if (n < p.N) {
            if (p.out_bf16) {
              __nv_bfloat162 lo = __floats2bfloat162_rn(o[0], o[1]), hi = __floats2bfloat162_rn(o[2], o[3]);
              *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + where) =
                  make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
            } else {
              *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + where) = make_float4(o[0], o[1], o[2], o[3]);
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (n + k < p.N) {
              if (p.out_bf16) reinterpret_cast<__nv_bfloat16*>(p.out)[where + k] = __float2bfloat16_rn(o[k]);
              else reinterpret_cast<float*>(p.out)[where + k] = o[k];
            }
        }
      }
    }
  }
  if constexpr (S > 1) {
    __syncwarp();
    cluster_sync_all();   // the others may still be reading this CTA's sums
  }
  __syncthreads();
  if (*abort_flag) {       // copies that nobody waited for may still be on their way
    for (int i = 0; i < 20; ++i) __nanosleep(1000);
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, F::kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres) != cudaSuccess ||
        qres != cudaDriverEntryPointSuccess)
      sym = nullptr;
    return reinterpret_cast<EncodeTiledFn>(sym);
  }();
  return fn;
}

// (rows, cols) matrix with a row pitch in bytes, read or written in boxes of 128 bytes x box_rows, 128-byte swizzle
int make_map(CUtensorMap* map, CUtensorMapDataType dt, int elem, const void* ptr, int64_t rows, int64_t cols, int64_t pitch,
             int box_rows) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return fail(TCFP_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / elem), (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(map, dt, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(TCFP_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
  return TCFP_OK;
}

// raises a kernel's dynamic shared memory limit, once for each device
template <typename Kernel>
int allow_smem(Kernel kern, int bytes, bool (&done)[64]) {
  int dev = 0;
  CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return fail(TCFP_ERR_UNSUPPORTED, "device index %d out of range", dev);
  if (!done[dev]) {
    CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done[dev] = true;
  }
  return TCFP_OK;
}

constexpr int kSmemLimit = 232448;       // of a block
constexpr int kSmemSm = 233472;          // of an SM; 1 KB of it goes with every block

// A block of the few-token kernel lets the next kernel's blocks in before it has its columns of TMEM, and those wait for it with
// theirs: whatever shares an SM has to fit into its 512 columns together.  A pair's block, which takes all of them, never fits
// beside a few-token block's shared memory, and as many of those as do fit stay below 512: none has more columns for its shared
// memory than the 128-token form, three of which have 384.
constexpr int kTmemColumns = 512;
static_assert(kPairSmem + 1024 + Few<16>::smem(Few<16>::kMinStages) + 1024 > kSmemSm, "a pair's block beside a few-token block");
template <int NT>
constexpr bool few_fit_tmem() {
  return kSmemSm / (Few<NT>::smem(Few<NT>::kMinStages) + 1024) * (int)Few<NT>::kTmemCols <= kTmemColumns;
}
static_assert(few_fit_tmem<16>() && few_fit_tmem<32>() && few_fit_tmem<64>() && few_fit_tmem<128>(), "few-token blocks of an SM");

struct Operands {
  const int8_t *a, *b;
  int64_t lda, ldb;
};

template <bool OUT_BF16, int G>
int launch_pair(const Operands& o, Int8Params p, cudaStream_t stream) {
  constexpr int kElem = OUT_BF16 ? 2 : 4;
  CUtensorMap tm_a, tm_b, tm_out;
  int rc;
  if ((rc = make_map(&tm_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, o.a, p.M, p.K, o.lda, 128)) != TCFP_OK) return rc;
  if ((rc = make_map(&tm_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, o.b, p.N, p.K, o.ldb, 128)) != TCFP_OK) return rc;
  const int64_t pitch = (int64_t)p.N * kElem;
  const int tma_store = pitch % 16 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0;
  tm_out = tm_a;
  if (tma_store && (rc = make_map(&tm_out, OUT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, kElem,
                                  p.out, p.M, p.N, pitch, 128)) != TCFP_OK)
    return rc;
  static bool done[64] = {false};
  if ((rc = allow_smem(int8_pair_kernel<OUT_BF16, G>, kPairSmem, done)) != TCFP_OK) return rc;
  p.group_m = 16;
  const int64_t tiles = (int64_t)((p.M + 255) / 256) * ((p.N + 255) / 256);
  const int max_pairs = gemm_sm_budget() / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * (tiles < max_pairs ? tiles : max_pairs)), 1, 1);
  cfg.blockDim = dim3(64 + 128 * G, 1, 1);
  cfg.dynamicSmemBytes = kPairSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {2, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  allow_early_start(cfg);
  CUDA_TRY(cudaLaunchKernelEx(&cfg, int8_pair_kernel<OUT_BF16, G>, tm_a, tm_b, tm_out, p, tma_store));
  return TCFP_OK;
}

template <int NT, int S>
int launch_few(const Operands& o, const Int8Params& p, cudaStream_t stream) {
  CUtensorMap tm_w, tm_x;
  int rc;
  if ((rc = make_map(&tm_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, o.b, p.N, p.K, o.ldb, 128)) != TCFP_OK) return rc;
  if ((rc = make_map(&tm_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, o.a, p.M, p.K, o.lda, NT)) != TCFP_OK) return rc;
  static bool done[64] = {false};
  if ((rc = allow_smem(int8_few_kernel<NT, S>, kSmemLimit, done)) != TCFP_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(S, (unsigned)((p.N + 127) / 128), (unsigned)((p.M + NT - 1) / NT));
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = Few<NT>::smem(p.stages);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {S, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  allow_early_start(cfg);
  CUDA_TRY(cudaLaunchKernelEx(&cfg, int8_few_kernel<NT, S>, tm_w, tm_x, p));
  return TCFP_OK;
}

// Splits of K: while the weight tiles alone leave SMs without work.  Measured (us, N x K, tokens: 1, 2, 4, 8 splits):
// 4096 x 4096, 1: 11.7, 8.3, 6.7, 6.8; 32: 12.1, 8.7, 7.5, 9.2.  12288 x 4096, 1: 14.5, 13.2, 12.0, 14.7; 64: 16.7, 15.2, 15.3,
// 22.2.  22016 x 4096, 1: 19.3, 19.4, 20.3, 24.8.  4096 x 11008, 1: 27.3, 16.8, 12.6, 10.9.  So up to three blocks an SM with
// 16 tokens, one and a half with more, whose sums take longer to join.
template <int NT>
int launch_few(const Operands& o, Int8Params p, cudaStream_t stream) {
  using F = Few<NT>;
  const int64_t tiles = (int64_t)((p.N + 127) / 128) * ((p.M + NT - 1) / NT);
  const int64_t room = (int64_t)sm_count() * (NT == 16 ? 6 : 3) / 2;
  int splits = 1;
  while (splits < 8 && 2 * splits * tiles <= room && 4 * splits <= p.k_stages) splits *= 2;
  // as many stages as the blocks that share an SM leave room for
  const int64_t blocks = tiles * splits;
  const int share = blocks <= sm_count() ? 1 : blocks <= 2 * sm_count() || NT == 128 ? 2 : 3;
  const int bytes = kSmemSm / share - 1024;
  int stages = ((bytes < kSmemLimit ? bytes : kSmemLimit) - F::smem(0)) / F::kStageBytes;
  const int need = (p.k_stages + splits - 1) / splits;
  stages = stages > need ? need : stages;
  p.stages = stages > kMaxFewStages ? kMaxFewStages : stages < F::kMinStages ? F::kMinStages : stages;
  switch (splits) {
    case 8: return launch_few<NT, 8>(o, p, stream);
    case 4: return launch_few<NT, 4>(o, p, stream);
    case 2: return launch_few<NT, 2>(o, p, stream);
    default: return launch_few<NT, 1>(o, p, stream);
  }
}

constexpr int64_t kMaxK = 131071;   // 128 * 128 * K stays below 2^31

}  // namespace
}  // namespace tcfp

using namespace tcfp;

extern "C" int32_t tcfp_int8_gemm(const int8_t* a, int64_t ld_a, const float* s_a, const int8_t* b, int64_t ld_b,
                                  const float* s_b, const float* bias, void* out, int32_t out_dtype, int64_t M, int64_t N,
                                  int64_t K, void* stream_) {
  const char* what = "tcfp_int8_gemm";
  cudaStream_t stream = (cudaStream_t)stream_;
  if (!a || !b || !s_a || !s_b || !out) return fail(TCFP_ERR_INVALID, "%s: NULL argument", what);
  if (out_dtype != TCFP_F32 && out_dtype != TCFP_BF16) return fail(TCFP_ERR_INVALID, "%s: out dtype %d", what, out_dtype);
  if (M < 1 || N < 1 || K < 1) return fail(TCFP_ERR_INVALID, "%s: M %lld, N %lld, K %lld", what, (long long)M, (long long)N, (long long)K);
  // tile indices in 32 bits, weight tiles in gridDim.y
  if (M > (1 << 30) || N > 65535 * 128) return fail(TCFP_ERR_UNSUPPORTED, "%s: M %lld, N %lld", what, (long long)M, (long long)N);
  if (K > kMaxK) return fail(TCFP_ERR_UNSUPPORTED, "%s: K %lld above %lld could overflow the integer sum", what, (long long)K, (long long)kMaxK);
  if (ld_a < K || ld_b < K || ld_a % 16 || ld_b % 16 || (reinterpret_cast<uintptr_t>(a) & 15u) || (reinterpret_cast<uintptr_t>(b) & 15u))
    return fail(TCFP_ERR_INVALID, "%s: rows of a and b start on 16-byte boundaries, ld >= K", what);
  const Operands o{a, b, ld_a, ld_b};
  Int8Params p{};
  p.s_a = s_a; p.s_b = s_b; p.bias = bias; p.out = out;
  p.M = (int)M; p.N = (int)N; p.K = (int)K;
  p.k_stages = (int)((K + kStageK - 1) / kStageK);
  p.out_bf16 = out_dtype == TCFP_BF16;
  p.status = device_status_ptr();
  p.wide_out = N % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
  // Tokens a tile: all of them up to 64; beyond, 64 while that leaves no SM two tiles, else 128.  The pairs take over where
  // tiles of 128 would not all be resident (two an SM), or would share SMs while the pairs need one tile each.  Measured
  // (us, few / pairs): 4096 x 4096, 256 tokens 11.6 / 16.8, 512: 13.6 / 17.2, 640: 17.9 / 16.9; 12288 x 4096, 128: 16.8 / 19.3,
  // 384: 21.1 / 28.1, 512: 35.8 / 28.5; 22016 x 4096, 128: 23.7 / 31.5, 256: 39.1 / 32.1; 1024 x 1024, 1024: 6.9 / 10.1.
  const int64_t rows = (N + 127) / 128, tiles = rows * ((M + 127) / 128), pair_tiles = ((N + 255) / 256) * ((M + 255) / 256);
  if (M > 64 && tiles > sm_count() && (tiles > 2 * sm_count() || 2 * pair_tiles <= sm_count())) {
    // From K = 2048 on a tile's K loop hides the epilogue of the tile before; for shorter ones two groups write it out.
    // Measured (us, one / two groups): 8192 x 12288 x 256 106 / 82, x 1024 110 / 97, x 4096 248 / 252.
    if (K < 2048) return p.out_bf16 ? launch_pair<true, 2>(o, p, stream) : launch_pair<false, 2>(o, p, stream);
    return p.out_bf16 ? launch_pair<true, 1>(o, p, stream) : launch_pair<false, 1>(o, p, stream);
  }
  if (M <= 16) return launch_few<16>(o, p, stream);
  if (M <= 32) return launch_few<32>(o, p, stream);
  if (M <= 64 || rows * ((M + 63) / 64) <= sm_count()) return launch_few<64>(o, p, stream);
  return launch_few<128>(o, p, stream);
}
