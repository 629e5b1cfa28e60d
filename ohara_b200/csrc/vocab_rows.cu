// Row operators over the vocabulary: log-probabilities of given tokens with entropies and the most
// likely alternatives, the distillation loss against a teacher's top tokens, and the gradients of
// both with respect to the logits.
//
// With z = x / T, m = max x, d = (x - m) / T, s = sum exp(d), q = exp(d) / s:
//   log-probability   l_t = d_t - log s
//   entropy           H   = log s - (sum exp(d) d) / s
//   top K             the K largest logits in order, ties to the lowest index
//   distillation      L   = sum_k p_k (log p_k - l_{i_k}) [+ p' (log p' - log q')]
// where p is the teacher's list (renormalised, or as it is with the rest p' = 1 - sum p in a bucket of
// its own against q' = sum of q over the tokens that are not listed). The statistics are (m, s) and
// not m + log s: for a row of the type's lowest value the sum would absorb log s.
//
// What bounds it: one read of the logits (forward), one read and one write (gradient); at bf16 the
// forward also needs the exponential unit for 73 % of the copy time. So a row is read once, 16 bytes per
// load and several loads in flight per thread; maximum, sum, entropy sum and the candidates for the
// top K are kept in registers as the row passes (a running maximum rescales the sums when it rises).
// A row is one CTA's work when there are many rows, and is cut over a cluster of two to eight CTAs
// when there are few; those join through the first CTA's shared memory, so no workspace is shared
// between calls and nothing depends on the order in which CTAs finish.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "api.h"
#include "common.cuh"
#include "host_utils.h"

namespace ob {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// A teacher's mass outside its list of up to this much is the rounding of the list's sum (K terms of
// relative error 2^-24 and the teacher's own) and counts as none: the student may have no token there.
constexpr float kLeastRest = 1e-6f;
constexpr int kUnroll = 4;       // 16-byte loads in flight per thread
constexpr int kMaxCluster = 8;   // the portable cluster size

// ---------------------------------------------------------------------------------------------
// Elements
// ---------------------------------------------------------------------------------------------
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
  static __device__ __forceinline__ void unpack(const uint4& r, float (&f)[4]) {
    f[0] = __uint_as_float(r.x), f[1] = __uint_as_float(r.y);
    f[2] = __uint_as_float(r.z), f[3] = __uint_as_float(r.w);
  }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void unpack(const uint4& r, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <>
struct Elem<__half> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
  static __device__ __forceinline__ void unpack(const uint4& r, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x, f[2 * i + 1] = v.y;
    }
  }
};

// N consecutive outputs in one store (8 or 16 bytes).
__device__ __forceinline__ void store_vec(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
}
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]),
                                            pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store_vec(__half* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_half(v[0], v[1]), pack_half(v[2], v[3]),
                                            pack_half(v[4], v[5]), pack_half(v[6], v[7]));
}

// Maximum that keeps a NaN (fmaxf drops it, and a NaN logit has to reach the top list).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ---------------------------------------------------------------------------------------------
// Order of the top list: value descending (NaN first, -0 equal to +0), then index ascending, as one
// unsigned 64-bit number. No element maps to 0.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint64_t rank_code(float x, uint32_t index) {
  const uint32_t b = __float_as_uint(x + 0.f);
  uint32_t key = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  if (x != x) key = 0xffffffffu;
  return (static_cast<uint64_t>(key) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ float code_value(uint64_t code) {
  const uint32_t key = static_cast<uint32_t>(code >> 32);
  if (key == 0xffffffffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
__device__ __forceinline__ uint32_t code_index(uint64_t code) {
  return 0xffffffffu - static_cast<uint32_t>(code);
}

// ---------------------------------------------------------------------------------------------
// Running statistics of the softmax of scaled logits (c = log2(e) / T): `m` the maximum seen (-inf:
// nothing finite yet), `s` the sum of e = 2^((x - m) c), and `w` by kind
//   kSum      nothing
//   kEntropy  the sum of e (x - m)
//   kSplit    the sum of e over the tokens outside the teacher's list; `s` is the sum inside it
// ---------------------------------------------------------------------------------------------
enum Kind { kSum, kEntropy, kSplit };

struct Stats {
  float m, s, w;
};

__device__ __forceinline__ float reference_of(float m) { return m == -INFINITY ? 0.f : m; }

// Moves the sums from maximum `a.m` to `m` (>= a.m).
template <Kind K>
__device__ __forceinline__ void rebase(Stats& a, float m, float c) {
  if (m == a.m) return;
  const float shift = a.m - m;  // < 0; -inf while nothing was seen or where the gap overflows
  const float f = fast_exp2(shift * c);
  if (f == 0.f) {
    // an empty or vanished sum becomes zero (0 * inf below would not), a NaN stays
    a.s = a.s == a.s ? 0.f : a.s;
    if (K != kSum) a.w = a.w == a.w ? 0.f : a.w;
  } else {
    if (K == kEntropy) a.w = f * fmaf(a.s, shift, a.w);
    if (K == kSplit) a.w *= f;
    a.s *= f;
  }
  a.m = m;
}

template <Kind K>
__device__ __forceinline__ void merge(Stats& a, Stats b, float c) {
  const float m = fmaxf(a.m, b.m);
  rebase<K>(a, m, c);
  rebase<K>(b, m, c);
  a.s += b.s;
  a.w += b.w;
}

// One logit, with the maximum already at or above it.
template <Kind K>
__device__ __forceinline__ void add_one(Stats& a, float x, float ref, float c, bool in_list = false) {
  const float d = x - ref;
  const float e = fast_exp2(d * c);
  if (K == kSplit && !in_list)
    a.w += e;
  else
    a.s += e;
  // a masked logit has e = 0 and d = -inf: the clamp makes their product 0 instead of NaN
  if (K == kEntropy) a.w = fmaf(e, fmaxf(d, -3.0e38f), a.w);
}

template <Kind K>
__device__ __forceinline__ Stats warp_merge(Stats a, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stats b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.w = __shfl_xor_sync(0xffffffffu, a.w, o);
    merge<K>(a, b, c);
  }
  return a;
}

// The CTA's statistics, in every thread of warp 0. One barrier.
template <Kind K, int THREADS>
__device__ __forceinline__ Stats block_merge(Stats a, float c, float4* scratch) {
  a = warp_merge<K>(a, c);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = make_float4(a.m, a.s, a.w, 0.f);
  __syncthreads();
  if (threadIdx.x < 32) {
    a = Stats{-INFINITY, 0.f, 0.f};
    if (threadIdx.x < THREADS / 32) {
      const float4 v = scratch[threadIdx.x];
      a = Stats{v.x, v.y, v.z};
    }
    a = warp_merge<K>(a, c);
  }
  return a;
}

// ---------------------------------------------------------------------------------------------
// Selection
// ---------------------------------------------------------------------------------------------
// The largest t such that exactly `k` codes of the CTA are >= t, found bit by bit with one barrier
// per bit; ends early once the count is exact. 1 (every code passes) when there are fewer than `k`.
// `count(t)` is this thread's number of codes >= t.
template <int THREADS, typename Count>
__device__ __forceinline__ uint64_t block_kth(int k, int (*partial)[THREADS / 32], Count count) {
  uint64_t prefix = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t cand = prefix | (1ull << bit);
    const int mine = __reduce_add_sync(0xffffffffu, count(cand));
    // two buffers: a warp writes one of them again only after the barrier of the other
    int* out = partial[bit & 1];
    if ((threadIdx.x & 31) == 0) out[threadIdx.x >> 5] = mine;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) total += out[i];
    if (total >= k) {
      prefix = cand;
      if (total == k) break;
    }
  }
  __syncthreads();
  return prefix == 0 ? 1 : prefix;
}

// ---------------------------------------------------------------------------------------------
// Geometry
// ---------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ const T* row_of(const RowsView& v, int64_t row) {
  const int64_t outer = row / v.inner;
  return static_cast<const T*>(v.base) + outer * v.outer_stride + (row - outer * v.inner) * v.inner_stride;
}

// A row as [head | vectors of N from a 16-byte boundary | tail]; the vectors are cut over `parts`
// CTAs at multiples of 32, head and tail belong to the first.
struct Slice {
  int head, tail_begin, v0, v1;
};
template <typename T>
__device__ __forceinline__ Slice slice_of(const T* row, int vocab, int part, int parts) {
  constexpr int N = Elem<T>::kN;
  Slice s;
  s.head = min(vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
  const int vecs = (vocab - s.head) / N;
  s.tail_begin = s.head + vecs * N;
  const int per = ((vecs + parts - 1) / parts + 31) & ~31;
  s.v0 = min((int64_t)part * per, (int64_t)vecs);
  s.v1 = min((int64_t)s.v0 + per, (int64_t)vecs);
  return s;
}
// The one head or tail element of this thread (-1: none): at most 7 of each, in different warps.
__device__ __forceinline__ int edge_index(const Slice& s, int vocab, int part) {
  if (part != 0) return -1;
  const int t = threadIdx.x;
  if (t < s.head) return t;
  if (t >= 32 && t - 32 < vocab - s.tail_begin) return s.tail_begin + t - 32;
  return -1;
}

// The .aligned forms want whole warps.
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void store_cluster_u64(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void store_cluster_f4(uint32_t addr, const Stats& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.m), "f"(v.s),
               "f"(v.w), "f"(0.f)
               : "memory");
}
__device__ __forceinline__ void store_cluster_i32(uint32_t addr, int v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// The statistics of all CTAs of the cluster, in warp 0 of the first one. `slots` is a shared array
// of kMaxCluster entries; the cluster barrier also publishes what the caller stored to the first CTA
// before the call, and no CTA leaves before every store to the first one has landed.
template <Kind K>
__device__ __forceinline__ Stats cluster_merge(Stats mine, float c, float4* slots, int part, int parts) {
  if (threadIdx.x == 0) store_cluster_f4(map_to_cta(smem_u32(&slots[part]), 0), mine);
  cluster_arrive();
  cluster_wait();
  Stats a{-INFINITY, 0.f, 0.f};
  if (part == 0 && threadIdx.x < 32) {
    if (threadIdx.x < parts) {
      const float4 v = slots[threadIdx.x];
      a = Stats{v.x, v.y, v.z};
    }
    a = warp_merge<K>(a, c);
  }
  return a;
}

// ---------------------------------------------------------------------------------------------
// Token log-probabilities
// ---------------------------------------------------------------------------------------------
template <int THREADS>
struct TopShared {
  static constexpr int kCap = THREADS >= 256 ? 8 * THREADS : 16 * THREADS;
  uint64_t codes[kCap];                          // candidates of this CTA's slice
  uint64_t merged[kMaxCluster][kMaxAlternatives];  // sorted lists of the cluster's CTAs
  int merged_count[kMaxCluster];
  uint64_t sorted[kMaxAlternatives];
  int partial[2][THREADS / 32];
  int count;
};
struct NoShared {
  int unused;
};

// Appends a candidate; the count goes on past a full list, which is how the caller notices.
template <int THREADS>
__device__ __forceinline__ void push(TopShared<THREADS>& sh, uint64_t code) {
  const int at = atomicAdd(&sh.count, 1);
  if (at < TopShared<THREADS>::kCap) sh.codes[at] = code;
}

// Cuts the candidate list down to the `k` largest (all of them if there are fewer).
template <int THREADS>
__device__ __forceinline__ uint64_t keep_largest(TopShared<THREADS>& sh, int k) {
  constexpr int kPer = TopShared<THREADS>::kCap / THREADS;
  const int n = sh.count;
  uint64_t mine[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = i * THREADS + (int)threadIdx.x;
    mine[i] = at < n ? sh.codes[at] : 0;
  }
  const uint64_t least = block_kth<THREADS>(k, sh.partial, [&](uint64_t t) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) c += mine[i] >= t ? 1 : 0;
    return c;
  });
  // every thread holds its candidates in registers: the list can be rewritten
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (mine[i] >= least) push<THREADS>(sh, mine[i]);
  __syncthreads();
  return least;
}

template <typename T, int THREADS, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(THREADS)
token_logprobs_kernel(const RowsView view, const TokenLogprobsArgs p) {
  constexpr int N = Elem<T>::kN;
  using Shared = std::conditional_t<TOP, TopShared<THREADS>, NoShared>;
  __shared__ Shared sh;
  __shared__ float4 scratch[THREADS / 32];
  __shared__ float4 slots[kMaxCluster];
  const int parts = p.parts;
  const int part = parts > 1 ? (int)cluster_cta_rank() : 0;
  const int64_t row = parts > 1 ? (int64_t)(blockIdx.x / parts) : (int64_t)blockIdx.x;
  const int tid = threadIdx.x;
  const int vocab = p.vocab;
  const int top = p.top;
  const float c = p.inv_temperature * kLog2e;
  constexpr Kind K = ENTROPY ? kEntropy : kSum;

  const int64_t token = p.tokens != nullptr ? p.tokens[row] : 0;
  if (p.tokens != nullptr && token == p.ignore_index) {
    // a row without a token: nothing of it is read, everything it returns is empty
    if (part == 0) {
      if (tid == 0) {
        if (p.logprobs != nullptr) p.logprobs[row] = 0.f;
        if (ENTROPY) p.entropy[row] = 0.f;
        p.stats[row] = make_float4(0.f, INFINITY, 0.f, 0.f);
      }
      if (TOP)
        for (int i = tid; i < top; i += THREADS) {
          p.top_logprobs[row * top + i] = -INFINITY;
          p.top_tokens[row * top + i] = -1;
        }
    }
    return;
  }
  if (parts > 1) cluster_arrive();  // the first CTA has to run before anything is stored to it
  const T* x = row_of<T>(view, row);
  const Slice sl = slice_of(x, vocab, part, parts);
  float target = __uint_as_float(0x7fffffffu);  // an index outside the vocabulary has no probability
  if (part == 0 && tid == 0 && p.logprobs != nullptr && token >= 0 && token < vocab)
    target = Elem<T>::load(x + token);

  Stats st{-INFINITY, 0.f, 0.f};
  const int edge = edge_index(sl, vocab, part);
  float edge_x = -INFINITY;
  if (edge >= 0) {
    edge_x = Elem<T>::load(x + edge);
    st.m = fmaxf(st.m, edge_x);
    add_one<K>(st, edge_x, reference_of(st.m), c);
  }
  const uint4* body = reinterpret_cast<const uint4*>(x + sl.head);
  uint64_t least = 1;         // candidates have to reach this code
  float least_x = -INFINITY;  // its value, for the first test of a whole vector
  bool overflow = false;
  if constexpr (TOP) {
    if (tid == 0) sh.count = 0;
    __syncthreads();
  }
  bool first = true;
  // every thread takes part in every sweep (they hold barriers), also in one that is empty for it
  for (int base = sl.v0; base < sl.v1 || (TOP && first); base += THREADS * kUnroll) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = base + u * THREADS + tid;
      if (v < sl.v1) raw[u] = body[v];
    }
    float high[kUnroll];  // NaN-keeping maximum of each vector
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      high[u] = -INFINITY;
      if (base + u * THREADS + tid >= sl.v1) continue;
      float f[N];
      Elem<T>::unpack(raw[u], f);
      float vm = f[0];
#pragma unroll
      for (int i = 1; i < N; ++i) vm = TOP ? max_nan(vm, f[i]) : fmaxf(vm, f[i]);
      high[u] = vm;
      if (vm > st.m) rebase<K>(st, vm, c);
      const float ref = reference_of(st.m);
#pragma unroll
      for (int i = 0; i < N; ++i) add_one<K>(st, f[i], ref, c);
    }
    if constexpr (TOP) {
      if (first) {
        // The k-th largest of the threads' own maxima is a bound that at least k elements reach.
        uint64_t best = edge >= 0 ? rank_code(edge_x, edge) : 0;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int v = base + u * THREADS + tid;
          if (v >= sl.v1) continue;
          float f[N];
          Elem<T>::unpack(raw[u], f);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const uint64_t code = rank_code(f[i], sl.head + v * N + i);
            best = code > best ? code : best;
          }
        }
        least = block_kth<THREADS>(top, sh.partial, [&](uint64_t t) { return best >= t ? 1 : 0; });
        least_x = least == 1 ? -INFINITY : code_value(least);
        if (edge >= 0 && rank_code(edge_x, edge) >= least) push<THREADS>(sh, rank_code(edge_x, edge));
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int v = base + u * THREADS + tid;
        if (v >= sl.v1 || high[u] < least_x) continue;
        float f[N];
        Elem<T>::unpack(raw[u], f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint64_t code = rank_code(f[i], sl.head + v * N + i);
          if (code >= least) push<THREADS>(sh, code);
        }
      }
      __syncthreads();
      const int n = sh.count;
      __syncthreads();
      if (n > TopShared<THREADS>::kCap) {
        overflow = true;
        if (tid == 0) sh.count = 0;  // found again below
        __syncthreads();
      } else if (n > TopShared<THREADS>::kCap / 2) {
        least = keep_largest<THREADS>(sh, top);
        least_x = code_value(least);
      }
    }
    first = false;
  }

  if constexpr (TOP) {
    if (overflow) {
      // More elements of one sweep pass the bound than the list holds (rows in ascending order and
      // the like): find the k-th largest of the slice by counting, which reads it once per bit.
      const uint64_t edge_code = edge >= 0 ? rank_code(edge_x, edge) : 0;
      auto each = [&](auto&& f) {
        for (int v = sl.v0 + tid; v < sl.v1; v += THREADS) {
          float e[N];
          Elem<T>::unpack(body[v], e);
#pragma unroll
          for (int i = 0; i < N; ++i) f(rank_code(e[i], sl.head + v * N + i));
        }
        if (edge >= 0) f(edge_code);
      };
      least = block_kth<THREADS>(top, sh.partial, [&](uint64_t t) {
        int n = 0;
        each([&](uint64_t code) { n += code >= t ? 1 : 0; });
        return n;
      });
      if (tid == 0) sh.count = 0;
      __syncthreads();
      each([&](uint64_t code) {
        if (code >= least) push<THREADS>(sh, code);
      });
      __syncthreads();
    } else if (sh.count > top) {
      keep_largest<THREADS>(sh, top);
    }
    // order the survivors by counting the larger ones
    const int n = sh.count;
    if (tid < n) {
      const uint64_t mine = sh.codes[tid];
      int larger = 0;
      for (int i = 0; i < n; ++i) larger += sh.codes[i] > mine ? 1 : 0;
      sh.sorted[larger] = mine;
    }
    __syncthreads();
  }

  Stats all = block_merge<K, THREADS>(st, c, scratch);
  if (parts > 1) {
    cluster_wait();  // every CTA of the cluster has started
    if constexpr (TOP) {
      const int n = sh.count;
      if (tid == 0) store_cluster_i32(map_to_cta(smem_u32(&sh.merged_count[part]), 0), n);
      if (tid < n)
        store_cluster_u64(map_to_cta(smem_u32(&sh.merged[part][tid]), 0), sh.sorted[tid]);
    }
    all = cluster_merge<K>(all, c, slots, part, parts);
    if (part != 0) return;
  }
  // ---- the row's results, by the (first) CTA --------------------------------------------------
  const float ref = reference_of(all.m);
  const float log_s = logf(all.s);
  if (tid == 0) {
    if (p.logprobs != nullptr)
      p.logprobs[row] = fmaf(target - ref, p.inv_temperature, -log_s);
    const float h = log_s - all.w * p.inv_temperature / all.s;
    if (ENTROPY) p.entropy[row] = h;
    p.stats[row] = make_float4(ref, all.s, ENTROPY ? h : 0.f, 0.f);
    scratch[0] = make_float4(ref, log_s, 0.f, 0.f);
  }
  if constexpr (TOP) {
    __syncthreads();
    const float r = scratch[0].x, ls = scratch[0].y;
    auto emit = [&](int place, uint64_t code) {
      if (place >= top) return;
      p.top_logprobs[row * top + place] = fmaf(code_value(code) - r, p.inv_temperature, -ls);
      p.top_tokens[row * top + place] = (int64_t)code_index(code);
    };
    if (parts == 1) {
      if (tid < top) emit(tid, sh.sorted[tid]);
    } else {
      // an entry's place: its place in its own list plus the larger entries of each other list
      for (int e = tid; e < parts * kMaxAlternatives; e += THREADS) {
        const int from = e / kMaxAlternatives, i = e - from * kMaxAlternatives;
        if (i >= sh.merged_count[from]) continue;
        const uint64_t code = sh.merged[from][i];
        int place = i;
        for (int other = 0; other < parts; ++other) {
          if (other == from) continue;
          int lo = 0, hi = sh.merged_count[other];
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (sh.merged[other][mid] > code) lo = mid + 1; else hi = mid;
          }
          place += lo;
        }
        emit(place, code);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Distillation from a teacher's list
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ float block_sum(float v, float* scratch, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  float total = 0.f;
  for (int i = 0; i < warps; ++i) total += scratch[i];
  return total;
}
__device__ __forceinline__ float block_max(float v, float* scratch, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  float total = scratch[0];
  for (int i = 1; i < warps; ++i) total = fmaxf(total, scratch[i]);
  return total;
}

// One bit per logit of the slice marks the listed tokens, a byte per 16-byte vector, so that the sum
// over the others is formed without a subtraction (1 - sum of the listed q would cancel away exactly
// where the student agrees with the teacher).
template <typename T, int THREADS, bool TAIL>
__global__ void __launch_bounds__(THREADS)
distillation_kernel(const RowsView view, const DistillationArgs p) {
  constexpr int N = Elem<T>::kN;
  extern __shared__ uint32_t marks[];
  __shared__ float4 scratch[THREADS / 32];
  __shared__ float4 slots[kMaxCluster];
  __shared__ float reduce[THREADS / 32];
  __shared__ int64_t listed[kMaxAlternatives];
  const int parts = p.parts;
  const int part = parts > 1 ? (int)cluster_cta_rank() : 0;
  const int64_t row = parts > 1 ? (int64_t)(blockIdx.x / parts) : (int64_t)blockIdx.x;
  const int tid = threadIdx.x;
  const int vocab = p.vocab;
  const float c = p.inv_temperature * kLog2e;
  constexpr Kind K = TAIL ? kSplit : kSum;
  const T* x = row_of<T>(view, row);
  const Slice sl = slice_of(x, vocab, part, parts);

  // ---- the teacher's entries, one per thread ---------------------------------------------------
  int64_t token = -1;
  float value = -INFINITY;
  if (tid < p.top) {
    token = p.tokens[row * p.top + tid];
    value = p.teacher[row * p.top + tid];
    if (token < 0) value = -INFINITY;
  }
  const bool counts = TAIL ? token >= 0 : value != -INFINITY;
  if (__syncthreads_count(counts) == 0) {  // an empty list teaches nothing: the row is not read
    if (part == 0 && tid == 0) {
      p.loss[row] = 0.f;
      p.stats[row] = make_float4(0.f, INFINITY, 0.f, 0.f);
    }
    return;
  }
  if (parts > 1) cluster_arrive();
  const bool inside = token >= 0 && token < vocab;
  float picked = __uint_as_float(0x7fffffffu);  // a token outside the vocabulary: NaN
  if (inside && part == 0) picked = Elem<T>::load(x + token);
  if (TAIL) {
    for (int i = tid; i < (sl.v1 - sl.v0 + 3) / 4; i += THREADS) marks[i] = 0;
    if (tid < p.top) listed[tid] = token;
    __syncthreads();
    if (inside && token >= sl.head && token < sl.tail_begin) {
      const int v = ((int)token - sl.head) / N;
      const int bit = ((int)token - sl.head) - v * N;
      if (v >= sl.v0 && v < sl.v1)
        atomicOr(&marks[(v - sl.v0) >> 2], 1u << (8 * ((v - sl.v0) & 3) + bit));
    }
    __syncthreads();
  }
  const uint8_t* mark = reinterpret_cast<const uint8_t*>(marks);

  // ---- one pass over the logits ----------------------------------------------------------------
  Stats st{-INFINITY, 0.f, 0.f};
  const int edge = edge_index(sl, vocab, part);
  if (edge >= 0) {
    const float f = Elem<T>::load(x + edge);
    bool in_list = false;
    if (TAIL)
      for (int k = 0; k < p.top; ++k) in_list |= listed[k] == edge;
    st.m = fmaxf(st.m, f);
    add_one<K>(st, f, reference_of(st.m), c, in_list);
  }
  const uint4* body = reinterpret_cast<const uint4*>(x + sl.head);
  for (int base = sl.v0 + tid; base < sl.v1; base += THREADS * kUnroll) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (base + u * THREADS < sl.v1) raw[u] = body[base + u * THREADS];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = base + u * THREADS;
      if (v >= sl.v1) continue;
      float f[N];
      Elem<T>::unpack(raw[u], f);
      float vm = f[0];
#pragma unroll
      for (int i = 1; i < N; ++i) vm = fmaxf(vm, f[i]);
      if (vm > st.m) rebase<K>(st, vm, c);
      const float ref = reference_of(st.m);
      const uint32_t in_list = TAIL ? mark[v - sl.v0] : 0;
      if (in_list == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) add_one<K>(st, f[i], ref, c);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) add_one<K>(st, f[i], ref, c, (in_list >> i) & 1);
      }
    }
  }
  Stats all = block_merge<K, THREADS>(st, c, scratch);
  if (parts > 1) {
    cluster_wait();
    all = cluster_merge<K>(all, c, slots, part, parts);
    if (part != 0) return;
  }

  // ---- the row's loss, by the (first) CTA -------------------------------------------------------
  if (tid == 0) slots[0] = make_float4(reference_of(all.m), all.s, all.w, 0.f);
  __syncthreads();
  const float ref = slots[0].x, outside = slots[0].z;
  const float total = TAIL ? slots[0].y + outside : slots[0].y;
  const float log_s = logf(total);
  float weight, log_weight, extra = 0.f;
  if (TAIL) {
    weight = expf(value);
    log_weight = value;
  } else {
    const float high = block_max(value, reduce, THREADS / 32);
    const float mass = block_sum(expf(value - high), reduce, THREADS / 32);
    weight = expf(value - high) / mass;
    log_weight = value - high - logf(mass);
    extra = high + logf(mass);
  }
  const float term =
      weight == 0.f ? 0.f : weight * (log_weight - fmaf(picked - ref, p.inv_temperature, -log_s));
  float loss = block_sum(term, reduce, THREADS / 32);
  if (TAIL) {
    extra = block_sum(weight, reduce, THREADS / 32);
    const float rest = 1.f - extra;
    if (!(rest <= kLeastRest)) loss += rest * (logf(rest) - (logf(outside) - log_s));
  }
  if (tid == 0) {
    p.loss[row] = loss;
    // a NaN loss has a NaN gradient, also where it comes from a token outside the vocabulary
    p.stats[row] = make_float4(ref, loss == loss ? total : loss, extra, outside);
  }
}

// ---------------------------------------------------------------------------------------------
// Gradients
// ---------------------------------------------------------------------------------------------
// Both operators' gradients are  e (slope t + level)  with t = (x - m) c and e = 2^t for the tokens
// that no entry names, so one streaming pass writes that everywhere and, after a barrier, one thread
// per named token overwrites its element with the full sum (rounded once; a token that several entries
// name is written by the first of them with all their weights, so the order of nothing matters).
template <typename T, typename O, int THREADS, bool DISTILL>
__global__ void __launch_bounds__(THREADS)
vocab_grad_kernel(const RowsView view, const VocabGradArgs p) {
  constexpr int N = Elem<T>::kN;
  __shared__ float reduce[THREADS / 32];
  __shared__ int64_t entry_token[kMaxAlternatives + 1];
  __shared__ float entry_weight[kMaxAlternatives + 1];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / p.parts;
  const int part = (int)(blockIdx.x - row * p.parts);
  const int vocab = p.vocab;
  const float c = p.inv_temperature * kLog2e;
  const T* x = row_of<T>(view, row);
  O* out = static_cast<O*>(p.out) + row * p.out_pitch;
  const Slice sl = slice_of(x, vocab, part, p.parts);
  const int edge = edge_index(sl, vocab, part);
  const float4 st = p.stats[row];
  const float ref = st.x, total = st.y;

  // ---- the row's coefficients ------------------------------------------------------------------
  float slope = 0.f, level, level_named;  // `level_named`: for the tokens that an entry names
  int entries = 0;
  bool zero = total == INFINITY;  // the forward pass skipped this row
  if (!zero) {
    if constexpr (DISTILL) {
      const float g = p.grad[row] * p.inv_temperature;
      zero = g == 0.f;
      entries = p.top;
      float mass = 1.f, rest = 0.f;
      if (p.tail) {
        mass = st.z;
        rest = 1.f - mass <= kLeastRest ? 0.f : 1.f - mass;
        mass += rest;
      }
      level_named = g * mass / total;
      // without outside mass every unnamed token has e = 0
      level = (rest > 0.f && st.w > 0.f) ? g * (mass / total - rest / st.w) : level_named;
      if (!zero && tid < entries) {
        const int64_t token = p.tokens[row * p.top + tid];
        const float value = p.teacher[row * p.top + tid];
        entry_token[tid] = token;
        entry_weight[tid] = token < 0 ? 0.f : -g * expf(p.tail ? value : value - st.z);
      }
    } else {
      float g = 0.f, gh = 0.f, g_top = 0.f, any = 0.f;
      int64_t token = -1;
      if (p.grad != nullptr) {
        g = p.grad[row];
        token = p.tokens[row];
        if (g != 0.f && (token < 0 || token >= vocab)) g = __uint_as_float(0x7fffffffu);
      }
      if (p.grad_entropy != nullptr) gh = p.grad_entropy[row];
      entries = 1;
      if (p.grad_top != nullptr) {
        entries += p.top;
        float mine = 0.f;
        if (tid < p.top) {
          mine = p.grad_top[row * p.top + tid];
          entry_token[1 + tid] = p.top_tokens[row * p.top + tid];
          entry_weight[1 + tid] = mine * p.inv_temperature;
        }
        g_top = block_sum(mine, reduce, THREADS / 32);
        any = __syncthreads_or(mine != 0.f) ? 1.f : 0.f;
      }
      zero = g == 0.f && gh == 0.f && any == 0.f;
      if (tid == 0) {
        entry_token[0] = token;
        entry_weight[0] = g * p.inv_temperature;
      }
      const float inv = p.inv_temperature / total;
      level = level_named = -inv * (g + g_top + gh * (st.z - logf(total)));
      slope = -inv * gh * kLn2;
    }
  }
  if (zero) {  // also where the logits hold NaN: nothing of this row was asked for
    entries = 0;
    slope = level = 0.f;
  }

  // ---- every token -----------------------------------------------------------------------------
  auto value = [&](float f, float lv) {
    // e is 0 from t = -150 down; the clamp keeps `slope t` finite there (masked logits: t = -inf)
    const float t = fmaxf((f - ref) * c, -1.0e4f);
    return fast_exp2(t) * fmaf(slope, t, lv);
  };
  if (edge >= 0) Elem<O>::store(out + edge, zero ? 0.f : value(Elem<T>::load(x + edge), level));
  const uint4* body = reinterpret_cast<const uint4*>(x + sl.head);
  O* out_body = out + sl.head;
  const bool aligned = reinterpret_cast<uintptr_t>(out_body) % (N * sizeof(O)) == 0;
  for (int base = sl.v0 + tid; base < sl.v1; base += THREADS * kUnroll) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (!zero && base + u * THREADS < sl.v1) raw[u] = body[base + u * THREADS];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = base + u * THREADS;
      if (v >= sl.v1) continue;
      float f[N];
      if (zero) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = 0.f;
      } else {
        Elem<T>::unpack(raw[u], f);
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = value(f[i], level);
      }
      if (aligned) {
        store_vec(out_body + (int64_t)v * N, f);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) Elem<O>::store(out_body + (int64_t)v * N + i, f[i]);
      }
    }
  }
  if (entries == 0) return;

  // ---- the named tokens of this part -----------------------------------------------------------
  __syncthreads();
  if (tid < entries) {
    const int64_t token = entry_token[tid];
    bool mine = token >= 0 && token < vocab;
    if (mine) {
      const int64_t in_body = token - sl.head;
      if (token < sl.head || token >= sl.tail_begin)
        mine = part == 0;
      else
        mine = in_body >= (int64_t)sl.v0 * N && in_body < (int64_t)sl.v1 * N;
    }
    for (int j = 0; mine && j < tid; ++j) mine = entry_token[j] != token;
    if (mine) {
      float weight = entry_weight[tid];
      for (int j = tid + 1; j < entries; ++j)
        if (entry_token[j] == token) weight += entry_weight[j];
      Elem<O>::store(out + token, value(Elem<T>::load(x + token), level_named) + weight);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------------------------
// CTAs that share a row: one when the rows alone fill the machine, else as many (up to a portable
// cluster) as still leave every thread a 16-byte load.
int parts_for(int64_t rows, int vocab, int per_vector, int threads) {
  const int vecs = vocab / per_vector;
  int parts = 1;
  while (parts < kMaxCluster && rows * parts < 2 * device_sm_count() && vecs >= 2 * parts * threads)
    parts *= 2;
  return parts;
}

template <typename Kernel, typename Args>
void launch_rows(Kernel kernel, int64_t ctas, int cluster, int threads, size_t smem,
                 const RowsView& view, const Args& args, cudaStream_t stream) {
  OB_CHECK(ctas <= 0x7fffffffll, "too many rows for one launch");
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  config.gridDim = dim3((unsigned)ctas, 1, 1);
  config.blockDim = dim3((unsigned)threads, 1, 1);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = attr;
  config.numAttrs = cluster > 1 ? 1 : 0;
  OB_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, view, args));
  count_launch();
}

template <typename T, int THREADS>
void logprobs_launch(const RowsView& view, TokenLogprobsArgs& a, int64_t rows, cudaStream_t stream) {
  a.parts = parts_for(rows, a.vocab, Elem<T>::kN, THREADS);
  auto go = [&](auto kernel) {
    launch_rows(kernel, rows * a.parts, a.parts, THREADS, 0, view, a, stream);
  };
  const bool h = a.entropy != nullptr, t = a.top > 0;
  if (h && t) go(token_logprobs_kernel<T, THREADS, true, true>);
  if (h && !t) go(token_logprobs_kernel<T, THREADS, true, false>);
  if (!h && t) go(token_logprobs_kernel<T, THREADS, false, true>);
  if (!h && !t) go(token_logprobs_kernel<T, THREADS, false, false>);
}

template <typename T, int THREADS>
void distillation_launch(const RowsView& view, DistillationArgs& a, int64_t rows, cudaStream_t stream) {
  constexpr int N = Elem<T>::kN;
  a.parts = parts_for(rows, a.vocab, N, THREADS);
  if (!a.tail) {
    launch_rows(distillation_kernel<T, THREADS, false>, rows * a.parts, a.parts, THREADS, 0, view, a, stream);
    return;
  }
  const size_t marks = ((size_t)(a.vocab / N + a.parts - 1) / a.parts + 31) / 32 * 32;
  OB_CHECK(marks <= 200 * 1024, "distillation: vocabulary too large for the token marks of a row");
  auto kernel = distillation_kernel<T, THREADS, true>;
  if (marks > 40 * 1024) ensure_dynamic_smem((const void*)kernel, 200 * 1024);
  launch_rows(kernel, rows * a.parts, a.parts, THREADS, marks, view, a, stream);
}

template <typename T, typename O>
void grad_launch(const RowsView& view, VocabGradArgs& a, int64_t rows, bool distill, cudaStream_t stream) {
  constexpr int threads = 256;
  const int vecs = a.vocab / Elem<T>::kN;
  a.parts = 1;
  while (a.parts < 64 && rows * a.parts < 8 * device_sm_count() && vecs >= 2 * a.parts * threads)
    a.parts *= 2;
  if (distill)
    launch_rows(vocab_grad_kernel<T, O, threads, true>, rows * a.parts, 1, threads, 0, view, a, stream);
  else
    launch_rows(vocab_grad_kernel<T, O, threads, false>, rows * a.parts, 1, threads, 0, view, a, stream);
}

// Rows of up to this many bytes get a small CTA: a large one would leave most of its threads idle.
constexpr int64_t kSmallRowBytes = 16 * 1024;

}  // namespace

void token_logprobs(const RowsView& view, LogitType type, TokenLogprobsArgs args, int64_t rows,
                    cudaStream_t stream) {
  if (rows == 0) return;
  OB_CHECK(args.top >= 0 && args.top <= kMaxAlternatives && args.top <= args.vocab,
           "token_logprobs: bad number of alternatives");
  const bool small = (int64_t)args.vocab * (type == LogitType::F32 ? 4 : 2) <= kSmallRowBytes;
  switch (type) {
    case LogitType::F32:
      small ? logprobs_launch<float, 128>(view, args, rows, stream)
            : logprobs_launch<float, 512>(view, args, rows, stream);
      break;
    case LogitType::BF16:
      small ? logprobs_launch<__nv_bfloat16, 128>(view, args, rows, stream)
            : logprobs_launch<__nv_bfloat16, 512>(view, args, rows, stream);
      break;
    case LogitType::F16:
      small ? logprobs_launch<__half, 128>(view, args, rows, stream)
            : logprobs_launch<__half, 512>(view, args, rows, stream);
      break;
  }
}

void distillation_loss(const RowsView& view, LogitType type, DistillationArgs args, int64_t rows,
                       cudaStream_t stream) {
  if (rows == 0) return;
  OB_CHECK(args.top >= 1 && args.top <= kMaxAlternatives, "distillation: bad length of the teacher's list");
  const bool small = (int64_t)args.vocab * (type == LogitType::F32 ? 4 : 2) <= kSmallRowBytes;
  switch (type) {
    case LogitType::F32:
      small ? distillation_launch<float, 128>(view, args, rows, stream)
            : distillation_launch<float, 512>(view, args, rows, stream);
      break;
    case LogitType::BF16:
      small ? distillation_launch<__nv_bfloat16, 128>(view, args, rows, stream)
            : distillation_launch<__nv_bfloat16, 512>(view, args, rows, stream);
      break;
    case LogitType::F16:
      small ? distillation_launch<__half, 128>(view, args, rows, stream)
            : distillation_launch<__half, 512>(view, args, rows, stream);
      break;
  }
}

void vocab_grad(const RowsView& view, LogitType type, LogitType out_type, VocabGradArgs args,
                int64_t rows, bool distill, cudaStream_t stream) {
  if (rows == 0) return;
  OB_CHECK(args.top >= 0 && args.top <= kMaxAlternatives, "vocabulary gradient: too many entries");
  if (type == LogitType::F32 && out_type == LogitType::F32)
    grad_launch<float, float>(view, args, rows, distill, stream);
  else if (type == LogitType::F32 && out_type == LogitType::BF16)
    grad_launch<float, __nv_bfloat16>(view, args, rows, distill, stream);
  else if (type == LogitType::BF16 && out_type == LogitType::BF16)
    grad_launch<__nv_bfloat16, __nv_bfloat16>(view, args, rows, distill, stream);
  else if (type == LogitType::F16 && out_type == LogitType::F16)
    grad_launch<__half, __half>(view, args, rows, distill, stream);
  else
    OB_CHECK(false, "vocabulary gradient: unsupported types");
}

}  // namespace ob
