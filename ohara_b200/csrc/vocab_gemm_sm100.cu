// The output projection and what is taken from its logits in one kernel: softmax statistics of every
// row (forward) or the gradient with respect to the logits (backward), so that fp32 logits never leave
// the tensor memory.
//
// The logits are X = H W^T, H (M x K) hidden states, W (N x K) the projection, N the vocabulary. A CTA
// pair owns a 256 x 256 tile of X per step: TMA brings both operands in 64-wide k-blocks, the leader
// issues `tcgen05.mma.cta_group::2`, and each CTA's eight epilogue warps drain 128 rows from TMEM, a
// thread holding one row of 128 columns:
//   statistics  maximum m, s = sum 2^((x - m) c), and with it the entropy's sum or the split into
//               tokens inside and outside a teacher's list (c = log2(e) / T). They are written per row
//               and half tile; a small kernel joins the N / 128 of them. A thread has all its 128
//               logits before it needs the maximum, so nothing is rescaled inside a tile, and the
//               accumulator is handed back before the first exponential.
//   gradient    e (slope t + level) with t = (x - m) c, e = 2^t, rounded to bf16 (the operand type of
//               the two products that follow) and stored by TMA; the few tokens that an entry names
//               are overwritten afterwards from their own fp32 logits.
// The logits of named tokens are plain dot products of H and gathered rows of W, fp32 sums of exact
// products like the tensor cores'.
//
// What bounds it: at K = 768 the tensor pipe needs 6100 cycles per tile and CTA, the exponentials
// 2048; storing fp32 logits and reading them back would move 8 bytes per logit, as long as the
// product itself takes. Tiles are dealt in groups of eight row tiles, so that one pass over W serves
// 2048 rows.
//
// Measured on one B200 at 8188 x 768 x 50304 (633 GFLOP; 383 us at the measured burst rate): statistics
// with the entropy 485 us (456 with one accumulator per tile, see kSegment), gradient 470 us, joining 20 us,
// named logits 8. A whole step takes 2.2 ms; with fp32 logits in memory and the row kernels behind the
// product it took 3.6.
#include "api.h"
#include "common.cuh"
#include "host_utils.h"
#include "vocab_rows.cuh"

namespace ob {

namespace {

using namespace vocab;

constexpr int kTileM = 256, kTileN = 256, kBlockK = 64;
// k-blocks that one accumulator sums. The tensor core's running fp32 sum loses a little at every step,
// always in the same direction; for the statistics, sums of at most 512 terms are added in registers
// instead, rounded to nearest. Error of a distillation loss at K = 2008: 1.1e-6 with one accumulator,
// 2.5e-7 so. (The gradient is rounded to bf16 and has no use for it.)
constexpr int kSegment = 8;
constexpr int kHalfM = 128;             // rows per CTA of the pair
constexpr int kRowGroup = 8;            // row tiles that share a pass over the vocabulary
constexpr int kEpilogueWarps = 8;
constexpr int kProducerWarp = 8, kMmaWarp = 9;
constexpr int kThreads = 320;
constexpr int kStageBytes = 2 * kHalfM * kBlockK * 2;  // 128 rows of each operand

// kModeGradPair writes the gradient as a sum of two bf16 matrices, the second below the first.
enum Mode { kModeSum = kSum, kModeEntropy = kEntropy, kModeSplit = kSplit, kModeGrad, kModeGradPair };
__host__ __device__ constexpr bool is_grad(Mode m) { return m == kModeGrad || m == kModeGradPair; }

template <Mode MODE>
struct Layout {
  // the gradient needs two 4 KB staging buffers per epilogue warp
  static constexpr int kStages = is_grad(MODE) ? 5 : 6;
  static constexpr int kStaging = is_grad(MODE) ? kEpilogueWarps * 2 * 4096 : 0;
  static constexpr int kTotal = kStages * kStageBytes + kStaging + 256 + 1024;
};

struct Params {
  int M, N, K, m_tiles, n_tiles;
  int h_rows[2];          // rows of H that each CTA of the pair loads per step
  float c;
  int* status;
  float4* partial;        // [2 n_tiles][m_tiles * 256]: m, s, w
  const uint32_t* marks;  // split: [M][8 n_tiles], a bit per listed token
  const float4* coef;     // gradient: [M] reference, level, slope
};

// Tile order: groups of kRowGroup row tiles; inside a group the row tile runs fastest.
__device__ __forceinline__ void decode(const Params& p, int tile, int& mt, int& nt) {
  const int per_group = kRowGroup * p.n_tiles;
  const int group = tile / per_group;
  const int first = group * kRowGroup;
  const int rows = min(kRowGroup, p.m_tiles - first);
  const int r = tile - group * per_group;
  nt = r / rows;
  mt = first + (r - nt * rows);
}

template <Mode MODE>
__global__ void __launch_bounds__(kThreads, 1)
vocab_gemm_kernel(const __grid_constant__ CUtensorMap tmH, const __grid_constant__ CUtensorMap tmW,
                  const __grid_constant__ CUtensorMap tmD, const __grid_constant__ CUtensorMap tmRest,
                  const Params p) {
  using L = Layout<MODE>;
  constexpr int kStages = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* staging = smem + kStages * kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + L::kStaging);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + kStages;
  uint64_t* tmem_full = bars + 2 * kStages;
  uint64_t* tmem_empty = tmem_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const WaitCtx wctx{abort_flag, p.status};
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t cta_rank = cluster_cta_rank();
  const int total_tiles = p.m_tiles * p.n_tiles;
  const int first_tile = (int)(blockIdx.x >> 1), tile_step = (int)(gridDim.x >> 1);
  const int k_blocks = (p.K + kBlockK - 1) / kBlockK;
  const int segments = is_grad(MODE) ? 1 : (k_blocks + kSegment - 1) / kSegment;
  const int per_segment = (k_blocks + segments - 1) / segments;  // the last may be shorter, not empty

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], 2 * kEpilogueWarps);  // of both CTAs
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kProducerWarp && lane == 0) {
    prefetch_tmap(&tmH);
    prefetch_tmap(&tmW);
    if (is_grad(MODE)) prefetch_tmap(&tmD);
  }
  if (warp == kMmaWarp) {
    tmem_alloc_pair(tmem_slot, 2 * kTileN);
    tmem_relinquish_pair();
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();  // nothing may touch the peer's barriers before it has initialised them
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == kProducerWarp) {
    // ------------------------------- TMA producer: 128 rows of H and of W per CTA ---------------
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int tile = first_tile; tile < total_tiles && ok; tile += tile_step) {
        int mt, nt;
        decode(p, tile, mt, nt);
        const int h_row = mt * kTileM + (int)cta_rank * kHalfM;
        const int w_row = nt * kTileN + (int)cta_rank * kHalfM;
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          const int s = it % kStages;
          if (!mbar_wait(&empty_bar[s], ((it / kStages) & 1) ^ 1, wctx, kTimeoutEmptyBarrier)) {
            ok = false;
            break;
          }
          uint8_t* sh = smem + s * kStageBytes;
          // the leader's barrier counts the bytes of both CTAs
          const uint32_t full_addr = map_to_cta(smem_u32(&full_bar[s]), 0);
          if (cta_rank == 0)
            mbar_expect_tx(&full_bar[s], kStageBytes + (p.h_rows[0] + p.h_rows[1]) * kBlockK * 2);
          if (p.h_rows[cta_rank] > 0)
            tma_load_3d_pair(sh, &tmH, full_addr, kb * kBlockK, h_row, 0);
          tma_load_3d_pair(sh + kHalfM * kBlockK * 2, &tmW, full_addr, kb * kBlockK, w_row, 0);
        }
      }
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------- MMA issuer (the leader's) ----------------------------------
    if (lane == 0 && cta_rank == 0) {
      const uint32_t idesc = make_idesc_bf16(kTileM, kTileN, false, false);
      const SmemDesc desc_h = make_smem_desc_parts(smem_u32(smem), 16, 1024);
      const SmemDesc desc_w = make_smem_desc_parts(smem_u32(smem + kHalfM * kBlockK * 2), 16, 1024);
      uint32_t it = 0, acc_iter = 0;
      bool ok = true;
      for (int tile = first_tile; tile < total_tiles && ok; tile += tile_step) {
        for (int begin = 0; begin < k_blocks && ok; begin += per_segment, ++acc_iter) {
          const int end = min(begin + per_segment, k_blocks);
          const uint32_t acc = acc_iter & 1;
          if (!mbar_wait(&tmem_empty[acc], ((acc_iter >> 1) & 1) ^ 1, wctx, kTimeoutTmemEmpty)) {
            ok = false;
            break;
          }
          tcgen05_fence_after();
          const uint32_t tmem_acc = tmem_base + acc * kTileN;
          for (int kb = begin; kb < end; ++kb, ++it) {
            const int s = it % kStages;
            if (!mbar_wait(&full_bar[s], (it / kStages) & 1, wctx, kTimeoutFullBarrier)) {
              ok = false;
              break;
            }
            tcgen05_fence_after();
#pragma unroll
            for (int k = 0; k < kBlockK / 16; ++k)
              umma_bf16_ss_pair(tmem_acc, smem_desc_at(desc_h, s * kStageBytes + k * 32),
                                smem_desc_at(desc_w, s * kStageBytes + k * 32), idesc,
                                (kb > begin || k > 0) ? 1u : 0u);
            const uint32_t addr = smem_u32(&empty_bar[s]);  // frees the stage in both CTAs
            tcgen05_commit_pair(map_to_cta(addr, 0));
            tcgen05_commit_pair(map_to_cta(addr, 1));
          }
          if (!ok) break;
          const uint32_t addr = smem_u32(&tmem_full[acc]);
          tcgen05_commit_pair(map_to_cta(addr, 0));
          tcgen05_commit_pair(map_to_cta(addr, 1));
        }
      }
    }
  } else {
    // ------------------------------- Epilogue ----------------------------------------------------
    const int quarter = warp & 3, half = warp >> 2;
    uint32_t acc_iter = 0, store_iter = 0;
    bool ok = true;
    const uint64_t c2 = pair(p.c, p.c);
    for (int tile = first_tile; tile < total_tiles; tile += tile_step) {
      int mt, nt;
      decode(p, tile, mt, nt);
      const int row0 = mt * kTileM + (int)cta_rank * kHalfM + quarter * 32;
      const int row = row0 + lane;
      const int col0 = nt * kTileN + half * 128;
      uint4 words = make_uint4(0, 0, 0, 0);
      float4 coef = make_float4(INFINITY, 0.f, 0.f, 0.f);
      if (row < p.M) {
        if (MODE == kModeSplit)
          words = *reinterpret_cast<const uint4*>(p.marks + ((int64_t)row * p.n_tiles + nt) * 8 + half * 4);
        if (is_grad(MODE)) coef = p.coef[row];
      }
      uint32_t v[4][32];
#pragma unroll 1
      for (int segment = 0; segment < segments; ++segment, ++acc_iter) {
        const uint32_t acc = acc_iter & 1;
        if (!mbar_wait(&tmem_full[acc], (acc_iter >> 1) & 1, wctx, kTimeoutTmemFull)) {
          ok = false;
          break;
        }
        tcgen05_fence_after();
        const uint32_t taddr =
            tmem_base + acc * kTileN + half * 128 + (static_cast<uint32_t>(quarter * 32) << 16);
        if (is_grad(MODE) || segment == 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) tmem_ld_32x32(taddr + 32 * i, v[i]);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t more[16];
            tmem_ld_32x16(taddr + 16 * i, more);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              uint32_t& sum = v[i >> 1][16 * (i & 1) + j];
              sum = __float_as_uint(__uint_as_float(sum) + __uint_as_float(more[j]));
            }
          }
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&tmem_empty[acc]), 0));
      }
      if (!ok) break;

      if constexpr (!is_grad(MODE)) {
        const int cols = p.N - col0;  // columns of this half that exist
        if (cols < 128) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (32 * i + j >= cols) v[i][j] = 0xff800000u;  // -inf
        }
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 32; ++j) m = fmaxf(m, __uint_as_float(v[i][j]));
        const float ref = m == -INFINITY ? 0.f : m;
        const uint64_t ref2 = pair(-ref, -ref);
        uint64_t s2[2] = {0, 0}, w2[2] = {0, 0};  // two chains each
        const uint32_t word[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const int chain = (j >> 1) & 1;
            const uint64_t x = pair(__uint_as_float(v[i][j]), __uint_as_float(v[i][j + 1]));
            const uint64_t t = mul2(add2(x, ref2), c2);
            const float2 tt = both(t);
            const float2 e = make_float2(fast_exp2(tt.x), fast_exp2(tt.y));
            if (MODE == kModeSplit) {
              const bool a = (word[i] >> j) & 1, b = (word[i] >> (j + 1)) & 1;
              s2[chain] = add2(s2[chain], pair(a ? e.x : 0.f, b ? e.y : 0.f));
              w2[chain] = add2(w2[chain], pair(a ? 0.f : e.x, b ? 0.f : e.y));
            } else {
              s2[chain] = add2(s2[chain], pair(e.x, e.y));
            }
            if (MODE == kModeEntropy)  // the clamp keeps 0 * -inf (columns past N) at 0
              w2[chain] = fma2(pair(e.x, e.y), pair(fmaxf(tt.x, -1.0e4f), fmaxf(tt.y, -1.0e4f)),
                               w2[chain]);
          }
        }
        const float2 s = both(add2(s2[0], s2[1])), w = both(add2(w2[0], w2[1]));
        const float scale = MODE == kModeEntropy ? 1.f / p.c : 1.f;  // sum e (x - m), as the row kernels have it
        if (row < p.M)
          p.partial[(int64_t)(2 * nt + half) * ((int64_t)p.m_tiles * kTileM) + row] =
              make_float4(m, s.x + s.y, (w.x + w.y) * scale, 0.f);
      } else {
        const uint64_t ref2 = pair(-coef.x, -coef.x);
        const uint64_t level2 = pair(coef.y, coef.y), slope2 = pair(coef.z, coef.z);
        uint8_t* my_staging = staging + warp * 2 * 4096;
#pragma unroll
        for (int part = 0; part < 2; ++part) {  // 64 columns: 128 bytes a row
          if (col0 + 64 * part >= p.N) break;   // uniform over the warp
          auto next_buffer = [&] {
            uint8_t* buf = my_staging + (store_iter & 1) * 4096;
            ++store_iter;
            if (lane == 0) tma_store_wait_read<1>();
            __syncwarp();
            return buf;
          };
          auto send = [&](const CUtensorMap* map, uint8_t* buf) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (row0 < p.M) tma_store_3d(map, buf, col0 + 64 * part, row0, 0);
              tma_store_commit();
            }
          };
          uint32_t rest[MODE == kModeGradPair ? 32 : 1];
          uint8_t* buf = next_buffer();
#pragma unroll
          for (int q = 0; q < 8; ++q) {  // 16 bytes
            uint32_t packed[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int col = 64 * part + 8 * q + 2 * r;
              const uint64_t x = pair(__uint_as_float(v[col >> 5][col & 31]),
                                      __uint_as_float(v[col >> 5][(col & 31) + 1]));
              float2 t = both(mul2(add2(x, ref2), c2));
              // e is 0 from t = -150 down; the clamp keeps slope t finite (and drops NaN where the
              // reference is +inf: a row that nothing asks for gets zeros whatever its logits)
              t = make_float2(fmaxf(t.x, -1.0e4f), fmaxf(t.y, -1.0e4f));
              const uint64_t e = pair(fast_exp2(t.x), fast_exp2(t.y));
              const float2 d = both(mul2(e, fma2(slope2, pair(t.x, t.y), level2)));
              packed[r] = pack_bf16(d.x, d.y);
              if constexpr (MODE == kModeGradPair)
                rest[4 * q + r] = pack_bf16(d.x - __uint_as_float(packed[r] << 16),
                                            d.y - __uint_as_float(packed[r] & 0xffff0000u));
            }
            *reinterpret_cast<uint4*>(buf + lane * 128 + ((q ^ (lane & 7)) << 4)) =
                make_uint4(packed[0], packed[1], packed[2], packed[3]);
          }
          send(&tmD, buf);
          if constexpr (MODE == kModeGradPair) {
            buf = next_buffer();
#pragma unroll
            for (int q = 0; q < 8; ++q)
              *reinterpret_cast<uint4*>(buf + lane * 128 + ((q ^ (lane & 7)) << 4)) =
                  make_uint4(rest[4 * q], rest[4 * q + 1], rest[4 * q + 2], rest[4 * q + 3]);
            send(&tmRest, buf);
          }
        }
      }
    }
    if (is_grad(MODE) && lane == 0) tma_store_wait_all<0>();
  }

  // ------------------------------- Teardown ---------------------------------------------------
  if (*abort_flag) {
    // give copies in flight time to land before shared memory is released
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 1000000ull) __nanosleep(1000);
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();  // a CTA outlives every access of its peer
  if (warp == kMmaWarp) {
    tcgen05_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * kTileN);
  }
}

template <Mode MODE>
void launch_gemm(const CUtensorMap& h, const CUtensorMap& w, const CUtensorMap& d,
                 const CUtensorMap& rest, const Params& p, cudaStream_t stream) {
  using L = Layout<MODE>;
  auto kernel = vocab_gemm_kernel<MODE>;
  static int resident_by_device[64] = {0};
  int dev = 0;
  OB_CUDA_CHECK(cudaGetDevice(&dev));
  int& resident = resident_by_device[dev & 63];
  ensure_dynamic_smem((const void*)kernel, L::kTotal);
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  config.blockDim = dim3(kThreads, 1, 1);
  config.dynamicSmemBytes = L::kTotal;
  config.stream = stream;
  config.attrs = attr;
  config.numAttrs = 1;
  const int sms = device_sm_count();
  if (resident == 0) {
    config.gridDim = dim3(2 * (sms / 2), 1, 1);
    int clusters = 0;
    OB_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&clusters, kernel, &config));
    resident = std::max(1, std::min(clusters, sms / 2));
  }
  const int pairs = (int)std::min<long long>((long long)p.m_tiles * p.n_tiles, resident);
  config.gridDim = dim3(2 * pairs, 1, 1);
  OB_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, h, w, d, rest, p));
  count_launch();
}

// ---------------------------------------------------------------------------------------------
// Joining
// ---------------------------------------------------------------------------------------------
constexpr int kJoinWarps = 16;

template <Kind K>
__device__ __forceinline__ void merge(Stats& a, Stats b, float c) {
  const float m = fmaxf(a.m, b.m);
  rebase<K>(a, m, c);
  rebase<K>(b, m, c);
  a.s += b.s;
  a.w += b.w;
}

// Eight rows per CTA: a warp reads 128 bytes (eight rows) of four half tiles at a time, so that one
// row over a large vocabulary still spreads over the CTA (1024 halves: 16 steps). The order of the
// sums is fixed. The joined statistics are in `out` after the barrier inside.
constexpr int kJoinRows = 8;
template <Kind K>
__device__ __forceinline__ void join_rows(const float4* partial, int halves, int64_t pitch, int M,
                                          float c, Stats (*part)[kJoinRows], Stats* out) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane & (kJoinRows - 1);
  const int row = blockIdx.x * kJoinRows + r;
  Stats a{-INFINITY, 0.f, 0.f};
  if (row < M) {
#pragma unroll 4
    for (int i = warp * 4 + (lane >> 3); i < halves; i += kJoinWarps * 4) {
      const float4 v = partial[i * pitch + row];
      merge<K>(a, Stats{v.x, v.y, v.z}, c);
    }
  }
  auto over_lanes = [&](int from) {  // lanes that differ in bits from `from` up hold the same row
    for (int o = from; o < 32; o <<= 1) {
      Stats b;
      b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
      b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
      b.w = __shfl_xor_sync(0xffffffffu, a.w, o);
      merge<K>(a, b, c);
    }
  };
  over_lanes(kJoinRows);
  if (lane < kJoinRows) part[warp][r] = a;
  __syncthreads();
  if (warp == 0) {
    a = part[lane >> 3][r];
    for (int i = 4 + (lane >> 3); i < kJoinWarps; i += 4) merge<K>(a, part[i][r], c);
    over_lanes(kJoinRows);
    if (lane < kJoinRows) out[r] = a;
  }
  __syncthreads();
}

template <Kind K>
__global__ void __launch_bounds__(kJoinWarps * 32)
join_logprobs_kernel(const float4* partial, int halves, int64_t pitch, int M, const float* picked,
                     const TokenLogprobsArgs p) {
  __shared__ Stats part[kJoinWarps][kJoinRows];
  __shared__ Stats joined[kJoinRows];
  join_rows<K>(partial, halves, pitch, M, p.inv_temperature * kLog2e, part, joined);
  const int row = blockIdx.x * kJoinRows + threadIdx.x;
  if (threadIdx.x >= kJoinRows || row >= M) return;
  if (p.tokens != nullptr && p.tokens[row] == p.ignore_index) {
    if (p.logprobs != nullptr) p.logprobs[row] = 0.f;
    if (K == kEntropy) p.entropy[row] = 0.f;
    p.stats[row] = make_float4(0.f, INFINITY, 0.f, 0.f);
    return;
  }
  const Stats a = joined[threadIdx.x];
  const float ref = reference_of(a.m);
  const float log_s = logf(a.s);
  if (p.logprobs != nullptr) p.logprobs[row] = fmaf(picked[row] - ref, p.inv_temperature, -log_s);
  const float h = log_s - a.w * p.inv_temperature / a.s;
  if (K == kEntropy) p.entropy[row] = h;
  p.stats[row] = make_float4(ref, a.s, K == kEntropy ? h : 0.f, 0.f);
}

template <bool TAIL>
__global__ void __launch_bounds__(kJoinWarps * 32)
join_distillation_kernel(const float4* partial, int halves, int64_t pitch, int M, const float* picks,
                         const DistillationArgs p) {
  __shared__ Stats part[kJoinWarps][kJoinRows];
  __shared__ Stats joined[kJoinRows];
  join_rows<TAIL ? kSplit : kSum>(partial, halves, pitch, M, p.inv_temperature * kLog2e, part, joined);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kJoinRows + warp;
  if (warp < kJoinRows && row < M) {
    if (!list_counts(p, row)) {
      if (lane == 0) skip_row(p, row);
      return;
    }
    float value[kEntriesPerLane], picked[kEntriesPerLane];
#pragma unroll
    for (int i = 0; i < kEntriesPerLane; ++i) {
      const int k = lane + 32 * i;
      const bool there = k < p.top && p.tokens[row * p.top + k] >= 0;
      value[i] = there ? p.teacher[row * p.top + k] : -INFINITY;
      picked[i] = there ? picks[row * p.top + k] : quiet_nan();
    }
    const Stats a = joined[warp];
    finish_distillation<TAIL>(p, row, value, picked, reference_of(a.m), TAIL ? a.s + a.w : a.s, a.w);
  }
}

// ---------------------------------------------------------------------------------------------
// Logits of named tokens: four entries per warp, whose gathers are in flight together
// ---------------------------------------------------------------------------------------------
constexpr int kPicks = 4;

__global__ void __launch_bounds__(256)
pick_logits_kernel(const __nv_bfloat16* h, int64_t ldh, const __nv_bfloat16* w, int64_t ldw,
                   const int64_t* tokens, float* picked, int64_t entries, int per_row, int vocab, int K) {
  const int64_t first = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * kPicks;
  const int lane = threadIdx.x & 31;
  const uint4* a[kPicks];
  const uint4* b[kPicks];
  bool inside[kPicks];
  uint64_t sum[kPicks];
#pragma unroll
  for (int e = 0; e < kPicks; ++e) {
    const int64_t at = min(first + e, entries - 1);
    const int64_t token = tokens[at];
    inside[e] = token >= 0 && token < vocab;
    a[e] = reinterpret_cast<const uint4*>(h + (at / per_row) * ldh);
    b[e] = reinterpret_cast<const uint4*>(w + (inside[e] ? token : 0) * ldw);
    sum[e] = 0;
  }
  for (int i = lane; i < K / 8; i += 32) {
    uint4 x[kPicks], y[kPicks];
#pragma unroll
    for (int e = 0; e < kPicks; ++e) {
      x[e] = a[e][i];
      y[e] = b[e][i];
    }
#pragma unroll
    for (int e = 0; e < kPicks; ++e) {
      const uint32_t xs[4] = {x[e].x, x[e].y, x[e].z, x[e].w}, ys[4] = {y[e].x, y[e].y, y[e].z, y[e].w};
#pragma unroll
      for (int q = 0; q < 4; ++q)
        sum[e] = fma2(pair(__uint_as_float(xs[q] << 16), __uint_as_float(xs[q] & 0xffff0000u)),
                      pair(__uint_as_float(ys[q] << 16), __uint_as_float(ys[q] & 0xffff0000u)), sum[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < kPicks; ++e) {
    const float2 s = both(sum[e]);
    const float total = warp_sum(s.x + s.y);
    if (lane == 0 && first + e < entries) picked[first + e] = inside[e] ? total : quiet_nan();
  }
}

// A bit per listed token: words of a row are consecutive, 8 per column tile.
__global__ void __launch_bounds__(256)
mark_tokens_kernel(const int64_t* tokens, uint32_t* marks, int64_t entries, int per_row, int vocab,
                   int64_t words) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= entries) return;
  const int64_t token = tokens[e];
  if (token >= 0 && token < vocab)
    atomicOr(marks + (e / per_row) * words + (token >> 5), 1u << (token & 31));
}

// ---------------------------------------------------------------------------------------------
// Gradient: coefficients before the product, named tokens after it
// ---------------------------------------------------------------------------------------------
// coef[row] = reference, level, slope, level of named tokens (see `GradRow`); a row that nothing asks
// for has an infinite reference, which makes every element 0.
template <bool DISTILL>
__global__ void __launch_bounds__(256)
grad_coefficients_kernel(const VocabGradArgs p, float4* coef, int M) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= M) return;
  const GradRow g = grad_row<DISTILL>(p, row, 0.f, false);
  coef[row] = g.zero ? make_float4(INFINITY, 0.f, 0.f, 0.f)
                     : make_float4(g.ref, g.level, g.slope, g.level_named);
}

template <bool DISTILL>
__global__ void __launch_bounds__(256)
grad_named_kernel(const VocabGradArgs p, const float4* coef, const float* picked, __nv_bfloat16* out,
                  int64_t pitch, int M, int two) {
  const int per_row = DISTILL ? p.top : 1;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= (int64_t)M * per_row) return;
  const int64_t row = e / per_row;
  const int k = (int)(e - row * per_row);
  const int64_t* tokens = p.tokens + row * per_row;
  const int64_t token = tokens[k];
  const float4 g = coef[row];
  if (token < 0 || token >= p.vocab || g.x == INFINITY) return;
  // the first of several entries of one token writes for all
  bool first = true;
  float weight = entry_weight<DISTILL>(p, row, k);
  if (DISTILL) {
#pragma unroll 8
    for (int j = 0; j < per_row; ++j) {
      if (j == k || tokens[j] != token) continue;
      if (j < k) first = false;
      if (j > k) weight += entry_weight<DISTILL>(p, row, j);
    }
  }
  if (!first) return;
  const float t = grad_exponent(picked[e], g.x, p.inv_temperature * kLog2e);
  const float d = fast_exp2(t) * fmaf(g.z, t, g.w) + weight;
  const __nv_bfloat16 first_part = __float2bfloat16_rn(d);
  out[row * pitch + token] = first_part;
  if (two) out[(row + M) * pitch + token] = __float2bfloat16_rn(d - __bfloat162float(first_part));
}

// out = sum of the parts, in order; four elements a thread.
template <typename O>
__global__ void __launch_bounds__(256)
sum_parts_kernel(const float4* parts, O* out, int64_t quads, int count) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < quads; i += (int64_t)gridDim.x * 256) {
    float4 a = parts[i];
    for (int s = 1; s < count; ++s) {
      const float4 b = parts[s * quads + i];
      a.x += b.x, a.y += b.y, a.z += b.z, a.w += b.w;
    }
    if constexpr (sizeof(O) == 4)
      reinterpret_cast<float4*>(out)[i] = a;
    else
      reinterpret_cast<uint2*>(out)[i] = make_uint2(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w));
  }
}

}  // namespace

void sum_parts(const float* parts, void* out, bool out_f32, int64_t elements, int count,
               cudaStream_t stream) {
  OB_CHECK(elements % 4 == 0 && count >= 1, "sum_parts: bad sizes");
  const int64_t quads = elements / 4;
  if (quads == 0) return;
  const unsigned blocks = (unsigned)std::min<int64_t>((quads + 255) / 256, 8 * device_sm_count());
  if (out_f32)
    sum_parts_kernel<<<blocks, 256, 0, stream>>>((const float4*)parts, (float*)out, quads, count);
  else
    sum_parts_kernel<<<blocks, 256, 0, stream>>>((const float4*)parts, (__nv_bfloat16*)out, quads, count);
  OB_LAUNCH_CHECK();
}

// ---------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------
namespace {

struct Plan {
  CUtensorMap h, w;
  Params p;
};
Plan make_plan(const LinearHead& head, float inv_temperature) {
  OB_CHECK(head.M > 0 && head.N > 0 && head.K > 0 && head.K % 8 == 0, "vocabulary product: bad sizes");
  Plan plan = {};
  Params& p = plan.p;
  p.M = head.M;
  p.N = head.N;
  p.K = head.K;
  p.m_tiles = (head.M + kTileM - 1) / kTileM;
  p.n_tiles = (head.N + kTileN - 1) / kTileN;
  OB_CHECK((long long)p.m_tiles * p.n_tiles <= 0x3fffffffll, "vocabulary product: too many tiles");
  p.c = inv_temperature * kLog2e;
  p.status = status_ptr();
  // A single row tile with few rows loads only those (in whole swizzle atoms of eight) and leaves the
  // rest of the operand as it is: a row of the product depends on its own row of H alone, and the
  // others are not used. Rows past the end of H would be filled by the copy, which costs as much as
  // real ones (1 x 2048 x 50304: 109 us a call against 70 with 256 rows).
  p.h_rows[0] = std::min(kHalfM, (head.M + 7) / 8 * 8);
  p.h_rows[1] = head.M <= kHalfM ? 0 : kHalfM;
  make_tmap_3d(&plan.h, head.hidden, TmapDtype::BF16, (uint64_t)head.K, (uint64_t)head.M, 1, head.ldh, 0,
               kBlockK, (uint32_t)p.h_rows[0], TmapSwizzle::B128);
  make_tmap_3d(&plan.w, head.weight, TmapDtype::BF16, (uint64_t)head.K, (uint64_t)head.N, 1, head.ldw, 0,
               kBlockK, kHalfM, TmapSwizzle::B128);
  return plan;
}

void pick_logits(const LinearHead& head, const int64_t* tokens, float* picked, int per_row,
                 cudaStream_t stream) {
  const int64_t entries = (int64_t)head.M * per_row;
  pick_logits_kernel<<<(unsigned)((entries + 8 * kPicks - 1) / (8 * kPicks)), 256, 0, stream>>>(
      (const __nv_bfloat16*)head.hidden, head.ldh, (const __nv_bfloat16*)head.weight, head.ldw, tokens,
      picked, entries, per_row, head.N, head.K);
  OB_LAUNCH_CHECK();
}

}  // namespace

int64_t linear_head_halves(int vocab) { return 2 * (int64_t)((vocab + kTileN - 1) / kTileN); }
int64_t linear_head_rows(int64_t rows) { return (rows + kTileM - 1) / kTileM * kTileM; }
int64_t linear_head_mark_words(int vocab) { return 8 * (int64_t)((vocab + kTileN - 1) / kTileN); }

void linear_token_logprobs(const LinearHead& head, const TokenLogprobsArgs& args, float4* partial,
                           float* picked, cudaStream_t stream) {
  Plan plan = make_plan(head, args.inv_temperature);
  plan.p.partial = partial;
  const int64_t pitch = (int64_t)plan.p.m_tiles * kTileM;
  const int halves = 2 * plan.p.n_tiles;
  if (args.logprobs != nullptr) pick_logits(head, args.tokens, picked, 1, stream);
  const unsigned blocks = (unsigned)((head.M + kJoinRows - 1) / kJoinRows);
  if (args.entropy != nullptr) {
    launch_gemm<kModeEntropy>(plan.h, plan.w, plan.w, plan.w, plan.p, stream);
    join_logprobs_kernel<kEntropy><<<blocks, kJoinWarps * 32, 0, stream>>>(partial, halves, pitch,
                                                                          head.M, picked, args);
  } else {
    launch_gemm<kModeSum>(plan.h, plan.w, plan.w, plan.w, plan.p, stream);
    join_logprobs_kernel<kSum><<<blocks, kJoinWarps * 32, 0, stream>>>(partial, halves, pitch, head.M,
                                                                      picked, args);
  }
  OB_LAUNCH_CHECK();
}

void linear_distillation(const LinearHead& head, const DistillationArgs& args, float4* partial,
                         float* picked, uint32_t* marks, cudaStream_t stream) {
  Plan plan = make_plan(head, args.inv_temperature);
  plan.p.partial = partial;
  const int64_t pitch = (int64_t)plan.p.m_tiles * kTileM;
  const int halves = 2 * plan.p.n_tiles;
  pick_logits(head, args.tokens, picked, args.top, stream);
  const unsigned blocks = (unsigned)((head.M + kJoinRows - 1) / kJoinRows);
  if (args.tail) {
    const int64_t words = 8 * (int64_t)plan.p.n_tiles;
    const int64_t entries = (int64_t)head.M * args.top;
    OB_CUDA_CHECK(cudaMemsetAsync(marks, 0, (size_t)head.M * words * 4, stream));
    mark_tokens_kernel<<<(unsigned)((entries + 255) / 256), 256, 0, stream>>>(
        args.tokens, marks, entries, args.top, head.N, words);
    OB_LAUNCH_CHECK();
    plan.p.marks = marks;
    launch_gemm<kModeSplit>(plan.h, plan.w, plan.w, plan.w, plan.p, stream);
    join_distillation_kernel<true><<<blocks, kJoinWarps * 32, 0, stream>>>(partial, halves, pitch,
                                                                            head.M, picked, args);
  } else {
    launch_gemm<kModeSum>(plan.h, plan.w, plan.w, plan.w, plan.p, stream);
    join_distillation_kernel<false><<<blocks, kJoinWarps * 32, 0, stream>>>(partial, halves, pitch,
                                                                          head.M, picked, args);
  }
  OB_LAUNCH_CHECK();
}

void linear_vocab_grad(const LinearHead& head, const VocabGradArgs& args, bool distill, bool two,
                       const float* picked, float4* coef, cudaStream_t stream) {
  Plan plan = make_plan(head, args.inv_temperature);
  plan.p.coef = coef;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(const_cast<void*>(args.out.base));
  const int64_t pitch = args.out.inner_stride;
  CUtensorMap d, rest;
  auto map = [&](CUtensorMap* m, void* base) {
    make_tmap_3d(m, base, TmapDtype::BF16, (uint64_t)head.N, (uint64_t)head.M, 1, pitch, 0, 64, 32,
                 TmapSwizzle::B128);
  };
  map(&d, out);
  map(&rest, two ? out + head.M * pitch : out);
  const unsigned rows = (unsigned)((head.M + 255) / 256);
  const int64_t entries = (int64_t)head.M * (distill ? args.top : 1);
  const unsigned named = (unsigned)((entries + 255) / 256);
  if (distill)
    grad_coefficients_kernel<true><<<rows, 256, 0, stream>>>(args, coef, head.M);
  else
    grad_coefficients_kernel<false><<<rows, 256, 0, stream>>>(args, coef, head.M);
  OB_LAUNCH_CHECK();
  if (two)
    launch_gemm<kModeGradPair>(plan.h, plan.w, d, rest, plan.p, stream);
  else
    launch_gemm<kModeGrad>(plan.h, plan.w, d, rest, plan.p, stream);
  if (distill)
    grad_named_kernel<true><<<named, 256, 0, stream>>>(args, coef, picked, out, pitch, head.M, two);
  else if (args.grad != nullptr)
    grad_named_kernel<false><<<named, 256, 0, stream>>>(args, coef, picked, out, pitch, head.M, two);
  else
    return;
  OB_LAUNCH_CHECK();
}

}  // namespace ob
