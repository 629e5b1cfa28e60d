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
//
// Measured on one B200 at 8188 x 50304 bf16 (824 MB; 126 us at the copy rate): log-probabilities 124 us
// (6.6 TB/s), with entropies 127, with the best token 149, the 20 / 64 best 179 / 233; distillation 133,
// with the tail 159; gradients 257 (6.4 TB/s read and written) and 271. The first versions took 188, 213,
// 551, 886 / 1144, 221 and 304: two logits per instruction, one maximum per warp before sums move, CTAs
// of 128 threads and the top list from vector bounds (instead of a search by bits) made the difference.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "api.h"
#include "common.cuh"
#include "host_utils.h"
#include "vocab_rows.cuh"

namespace ob {

namespace {

using namespace vocab;

constexpr int kUnroll = 4;       // 16-byte loads in flight per thread
constexpr int kMaxCluster = 8;   // the portable cluster size

// Maximum that keeps a NaN (fmaxf drops it, and a NaN logit has to reach the top list).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

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
  static __device__ __forceinline__ float highest(const uint4& r) {
    return max_nan(max_nan(__uint_as_float(r.x), __uint_as_float(r.y)),
                   max_nan(__uint_as_float(r.z), __uint_as_float(r.w)));
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
  static __device__ __forceinline__ float highest(const uint4& r) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
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
  static __device__ __forceinline__ float highest(const uint4& r) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
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
// A thread's part of a row
// ---------------------------------------------------------------------------------------------
// A thread's sums over the logits it has read, even and odd elements apart.
struct Running {
  float m;
  uint64_t s, w;
};

template <Kind K>
__device__ __forceinline__ void raise(Running& a, float m, float c) {
  const float shift = a.m - m;
  const float f = fast_exp2(shift * c);
  if (f == 0.f) {  // as in `rebase`
    const float2 s = both(a.s), w = both(a.w);
    a.s = pair(s.x == s.x ? 0.f : s.x, s.y == s.y ? 0.f : s.y);
    a.w = pair(w.x == w.x ? 0.f : w.x, w.y == w.y ? 0.f : w.y);
  } else {
    const uint64_t f2 = pair(f, f);
    if (K == kEntropy) a.w = fma2(a.s, pair(shift, shift), a.w);
    if (K != kSum) a.w = mul2(a.w, f2);
    a.s = mul2(a.s, f2);
  }
  a.m = m;
}

// The N logits of one vector, with the maximum already at or above them. `in_list` (kSplit): a bit per
// logit. Per pair: subtract, scale, two exponentials, add (and clamp, fuse for the entropy).
template <Kind K, int N>
__device__ __forceinline__ void accumulate(Running& a, const float (&f)[N], float c, uint32_t in_list) {
  const float ref = reference_of(a.m);
  const uint64_t ref2 = pair(-ref, -ref), c2 = pair(c, c);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const uint64_t d = add2(pair(f[i], f[i + 1]), ref2);
    const float2 t = both(mul2(d, c2));
    const float2 e = make_float2(fast_exp2(t.x), fast_exp2(t.y));
    if (K == kSplit) {
      if (in_list == 0) {
        a.w = add2(a.w, pair(e.x, e.y));
      } else {
        const bool x = (in_list >> i) & 1, y = (in_list >> (i + 1)) & 1;
        a.s = add2(a.s, pair(x ? e.x : 0.f, y ? e.y : 0.f));
        a.w = add2(a.w, pair(x ? 0.f : e.x, y ? 0.f : e.y));
      }
    } else {
      a.s = add2(a.s, pair(e.x, e.y));
    }
    if (K == kEntropy) {
      const float2 dd = both(d);
      a.w = fma2(pair(e.x, e.y), pair(fmaxf(dd.x, -3.0e38f), fmaxf(dd.y, -3.0e38f)), a.w);
    }
  }
}

// The sums of one logit.
template <Kind K>
__device__ __forceinline__ Running first_of(float x, float c, bool in_list) {
  Running a{fmaxf(x, -INFINITY), 0, 0};  // a NaN is no maximum
  const float e = fast_exp2((x - reference_of(a.m)) * c);
  if (K == kSplit && !in_list)
    a.w = pair(e, 0.f);
  else
    a.s = pair(e, 0.f);
  return a;
}

__device__ __forceinline__ Stats folded(const Running& a) {
  const float2 s = both(a.s), w = both(a.w);
  return Stats{a.m, s.x + s.y, w.x + w.y};
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
  // (a 64-bit division is sixty instructions, and most views have one leading stride)
  const int64_t outer = row < v.inner ? 0 : row / v.inner;
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

// The statistics of all CTAs of the cluster, in every warp of the first one. `slots` is a shared array
// of kMaxCluster entries; the cluster barrier also publishes what the caller stored to the first CTA
// before the call, and no CTA leaves before every store to the first one has landed.
template <Kind K>
__device__ __forceinline__ Stats cluster_merge(Stats mine, float c, float4* slots, int part, int parts) {
  if (threadIdx.x == 0) store_cluster_f4(map_to_cta(smem_u32(&slots[part]), 0), mine);
  cluster_arrive();
  cluster_wait();
  Stats a{-INFINITY, 0.f, 0.f};
  const int lane = threadIdx.x & 31;
  if (part == 0 && lane < parts) {
    const float4 v = slots[lane];
    a = Stats{v.x, v.y, v.z};
  }
  return warp_merge<K>(a, c);
}

// ---------------------------------------------------------------------------------------------
// Token log-probabilities
// ---------------------------------------------------------------------------------------------
// The top K of a row without a second pass over it. Every lane remembers its best vector so far (its
// maximum and position); the j-th best of a warp's 32 lanes, and the i-th best of those over the warps
// (i j >= K), is a vector that at least K distinct vectors reach, so no element of a vector below
// that bound can be among the K. Vectors that reach it are noted (their position, in a list of the
// warp), the bound is taken again after 1, 2, 4, ... sweeps, and at the end the noted vectors are read
// once more (from L2) against the last bound. For random logits that leaves about 1.75 K elements, which
// are ordered by counting. The order of vectors is (maximum, then position), so ties - a row of one
// value, masked logits - do not flood the lists. A row that floods them all the same (in ascending
// order, say) goes through `block_kth` over the whole slice.
template <int THREADS>
struct TopShared {
  static constexpr int kWarps = THREADS / 32;
  static constexpr int kHits = THREADS == 512 ? 128 : 512;  // noted vectors of a warp
  static constexpr int kCap = THREADS == 128 ? 1024 : (THREADS == 256 ? 2048 : 2560);
  uint64_t codes[kCap];  // elements that reach the last bound
  uint32_t hits[kWarps][kHits];
  uint64_t bound[kWarps];  // of each warp, read by the others without a barrier: none ever gets invalid
  int partial[2][kWarps];
  int count, overflow;
};
// What joins the CTAs of a cluster (the 512-thread shape).
struct ClusterLists {
  uint64_t merged[kMaxCluster][kMaxAlternatives];
  int merged_count[kMaxCluster];
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
__device__ __forceinline__ void keep_largest(TopShared<THREADS>& sh, int k) {
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
}

// A vector's code: its maximum, then its position, ascending positions last. 16-bit logits need 16 bits
// for the maximum, which leaves 16 of a register for the position (in units of 2^shift vectors, 1 for
// vocabularies below 2^19): half the instructions of the general form. Two lanes whose codes are then
// equal only make the bound a little weaker.
template <typename T>
struct VectorCode {
  using Code = uint64_t;
  static __device__ __forceinline__ int shift_for(int) { return 0; }
  static __device__ __forceinline__ Code make(float x, int at) { return rank_code(x, (uint32_t)at); }
  static __device__ __forceinline__ float value(Code c) { return code_value(c); }
  static __device__ __forceinline__ int at(Code c) { return (int)code_index(c); }
};
__device__ __forceinline__ int code_shift16(int vecs) { return max(0, 16 - __clz(vecs)); }
template <>
struct VectorCode<__nv_bfloat16> {
  using Code = uint32_t;
  static __device__ __forceinline__ int shift_for(int vecs) { return code_shift16(vecs); }
  static __device__ __forceinline__ Code make(float x, int at) {
    return (static_cast<uint32_t>(rank_code(x, 0) >> 32) & 0xffff0000u) | (0xffffu - at);
  }
  static __device__ __forceinline__ float value(Code c) {
    const uint32_t key = c >> 16;
    if (key == 0xffffu) return __uint_as_float(0x7fffffffu);
    return __uint_as_float(((key & 0x8000u) ? (key & 0x7fffu) : (~key & 0xffffu)) << 16);
  }
  static __device__ __forceinline__ int at(Code c) { return 0xffff - (int)(c & 0xffffu); }
};
template <>
struct VectorCode<__half> {
  using Code = uint32_t;
  static __device__ __forceinline__ int shift_for(int vecs) { return code_shift16(vecs); }
  static __device__ __forceinline__ Code make(float x, int at) {
    const uint32_t b = __half_as_ushort(__float2half_rn(x + 0.f));  // exact: x was a half
    uint32_t key = (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u);
    if (x != x) key = 0xffffu;
    return (key << 16) | (0xffffu - at);
  }
  static __device__ __forceinline__ float value(Code c) {
    const uint32_t key = c >> 16;
    if (key == 0xffffu) return __uint_as_float(0x7fffffffu);
    const uint16_t b = (uint16_t)((key & 0x8000u) ? (key & 0x7fffu) : (~key & 0xffffu));
    return __half2float(__ushort_as_half(b));
  }
  static __device__ __forceinline__ int at(Code c) { return 0xffff - (int)(c & 0xffffu); }
};

// The n-th largest of the lanes' codes (0 where there are fewer), and the least.
__device__ __forceinline__ uint64_t warp_nth(uint64_t code, int n) {
  uint32_t hi = static_cast<uint32_t>(code >> 32), lo = static_cast<uint32_t>(code);
  uint32_t h = 0, l = 0;
  for (int i = 0; i < n; ++i) {
    h = __reduce_max_sync(0xffffffffu, hi);
    l = __reduce_max_sync(0xffffffffu, hi == h ? lo : 0u);
    if (hi == h && lo == l) hi = lo = 0;
  }
  return (static_cast<uint64_t>(h) << 32) | l;
}
__device__ __forceinline__ uint32_t warp_nth(uint32_t code, int n) {
  uint32_t most = 0;
  for (int i = 0; i < n; ++i) {
    most = __reduce_max_sync(0xffffffffu, code);
    if (code == most) code = 0;
  }
  return most;
}
__device__ __forceinline__ uint64_t warp_least(uint64_t code) {
  const uint32_t hi = static_cast<uint32_t>(code >> 32), lo = static_cast<uint32_t>(code);
  const uint32_t h = __reduce_min_sync(0xffffffffu, hi);
  const uint32_t l = __reduce_min_sync(0xffffffffu, hi == h ? lo : 0xffffffffu);
  return (static_cast<uint64_t>(h) << 32) | l;
}
__device__ __forceinline__ uint32_t warp_least(uint32_t code) {
  return __reduce_min_sync(0xffffffffu, code);
}

// How the bound for the K best is put together: the `per_warp`-th best lane of every warp, then the
// `of_warps`-th best of those.
struct BoundPlan {
  int per_warp, of_warps;
};
template <int THREADS>
__device__ __forceinline__ BoundPlan bound_plan(int top) {
  constexpr int kWarps = THREADS / 32;
  const int per_warp = (top + kWarps - 1) / kWarps;
  return BoundPlan{per_warp, (top + per_warp - 1) / per_warp};
}
template <int WARPS, typename Code>
__device__ __forceinline__ Code joint_bound(const volatile Code* bound, const BoundPlan& plan) {
  const int lane = threadIdx.x & 31;
  if (plan.of_warps == WARPS) return warp_least(lane < WARPS ? bound[lane] : ~Code(0));
  return warp_nth(lane < WARPS ? bound[lane] : Code(0), plan.of_warps);
}

template <typename T, int THREADS, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(THREADS, TOP ? (THREADS == 512 ? 2 : 1280 / THREADS) : (THREADS == 512 ? 3 : 1792 / THREADS))
token_logprobs_kernel(const RowsView view, const TokenLogprobsArgs p) {
  constexpr int N = Elem<T>::kN;
  constexpr int kWarps = THREADS / 32;
  constexpr bool CLUSTER = THREADS == 512;
  constexpr Kind K = ENTROPY ? kEntropy : kSum;
  __shared__ std::conditional_t<TOP, TopShared<THREADS>, NoShared> sh;
  __shared__ std::conditional_t<TOP && CLUSTER, ClusterLists, NoShared> joined;
  __shared__ float4 scratch[kWarps];
  __shared__ float4 slots[CLUSTER ? kMaxCluster : 1];
  const int parts = CLUSTER ? p.parts : 1;
  const int part = parts > 1 ? (int)cluster_cta_rank() : 0;
  const int64_t row = parts > 1 ? (int64_t)(blockIdx.x / parts) : (int64_t)blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int vocab = p.vocab;
  const int top = p.top;
  const float c = p.inv_temperature * kLog2e;

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

  Running run{-INFINITY, 0, 0};
  const int edge = edge_index(sl, vocab, part);
  float edge_x = -INFINITY;
  if (edge >= 0) {
    edge_x = Elem<T>::load(x + edge);
    run = first_of<K>(edge_x, c, false);
  }
  const uint4* body = reinterpret_cast<const uint4*>(x + sl.head);

  // the lane's best vector (NaN aside: that reaches every bound), the bound, and how many vectors
  // the warp has noted
  float best = -INFINITY, least_x = -INFINITY;
  int best_at = -1, least_at = 0x7fffffff, noted = 0, refresh_at = 0x7fffffff;
  const BoundPlan plan = TOP ? bound_plan<THREADS>(top) : BoundPlan{1, 1};
  using V = VectorCode<T>;
  using Code = typename V::Code;
  const int shift = V::shift_for(sl.v1);
  auto publish_bound = [&] {
    if constexpr (TOP) {
      const Code b = warp_nth(best_at < 0 ? Code(0) : V::make(best, best_at >> shift), plan.per_warp);
      if (lane == 0) reinterpret_cast<volatile Code*>(sh.bound)[warp] = b;
    }
  };
  auto take_bound = [&] {
    if constexpr (TOP) {
      const Code b = joint_bound<kWarps>(reinterpret_cast<const volatile Code*>(sh.bound), plan);
      least_x = b == 0 ? -INFINITY : V::value(b);
      least_at = b == 0 ? 0x7fffffff : (((V::at(b) + 1) << shift) - 1);
    }
  };
  if constexpr (TOP) {
    if (tid == 0) sh.count = sh.overflow = 0;
  }
  int sweep = 0;
  // kUnroll vectors per thread; a full sweep has all of them, which spares the tests
  auto one_sweep = [&](int base, auto full) {
    constexpr bool FULL = decltype(full)::value;
    auto there = [&](int u) { return FULL || base + u * THREADS + tid < sl.v1; };
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (there(u)) raw[u] = body[base + u * THREADS + tid];
    float high[kUnroll];  // NaN-keeping maximum of each vector
    float sweep_high = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      high[u] = there(u) ? Elem<T>::highest(raw[u]) : -INFINITY;
      sweep_high = fmaxf(sweep_high, high[u]);
      if (TOP) nan |= high[u] != high[u];
    }
    if (sweep_high > run.m) raise<K>(run, sweep_high, c);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (!there(u)) continue;
      float f[N];
      Elem<T>::unpack(raw[u], f);
      accumulate<K>(run, f, c, 0);
    }
    if constexpr (TOP) {
      if (sweep == 0 && there(0)) best_at = base + tid;  // also if that is -inf
      if (sweep_high > best) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          if (high[u] > best) {
            best = high[u];
            best_at = base + u * THREADS + tid;
          }
        }
      }
      // after 1, 2, 4, ... sweeps, and when many vectors were noted since the last time
      if ((sweep & (sweep + 1)) == 0 || noted >= refresh_at) {
        publish_bound();
        if (sweep == 0) __syncthreads(); else __syncwarp();
        take_bound();
        refresh_at = noted + 128;
      }
      if (__any_sync(0xffffffffu, nan || !(sweep_high < least_x))) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int v = base + u * THREADS + tid;
          const bool hit = there(u) && !(high[u] < least_x) && (high[u] != least_x || v <= least_at);
          const uint32_t mask = __ballot_sync(0xffffffffu, hit);
          if (mask == 0) continue;
          const int at = noted + __popc(mask & ((1u << lane) - 1));
          if (hit && at < TopShared<THREADS>::kHits) sh.hits[warp][at] = (uint32_t)v;
          noted += __popc(mask);
        }
      }
      ++sweep;
    }
  };
  int base = sl.v0;
  for (; base + THREADS * kUnroll <= sl.v1; base += THREADS * kUnroll)
    one_sweep(base, std::true_type{});
  // (a first sweep also where it is empty: it holds a barrier)
  if (base < sl.v1 || (TOP && sweep == 0)) one_sweep(base, std::false_type{});

  // ---- statistics of the CTA (in every warp) and the last bound: one barrier --------------------
  Stats all = warp_merge<K>(folded(run), c);
  if (lane == 0) scratch[warp] = make_float4(all.m, all.s, all.w, 0.f);
  publish_bound();
  if constexpr (TOP) {
    if (lane == 0 && noted > TopShared<THREADS>::kHits) sh.overflow = 1;
  }
  __syncthreads();
  all = Stats{-INFINITY, 0.f, 0.f};
  if (lane < kWarps) {
    const float4 v = scratch[lane];
    all = Stats{v.x, v.y, v.z};
  }
  all = warp_merge<K>(all, c);

  int found = 0;  // elements in `codes`, of which the `top` largest are the slice's list
  if constexpr (TOP) {
    take_bound();
    const uint64_t edge_code = edge >= 0 ? rank_code(edge_x, edge) : 0;
    if (sh.overflow == 0) {
      // an element reaches the bound if its vector could have: the last place of the bound's vector
      const uint64_t least =
          least_at >= sl.v1 ? (least_x == -INFINITY ? 1 : rank_code(least_x, vocab))
                            : rank_code(least_x, sl.head + least_at * N + N - 1);
      for (int i = lane; i < noted; i += 32) {
        const int v = (int)sh.hits[warp][i];
        float f[N];
        Elem<T>::unpack(body[v], f);
#pragma unroll
        for (int q = 0; q < N; ++q) {
          if (f[q] < least_x) continue;
          const uint64_t code = rank_code(f[q], sl.head + v * N + q);
          if (code >= least) push<THREADS>(sh, code);
        }
      }
      if (edge_code >= least) push<THREADS>(sh, edge_code);
    }
    __syncthreads();
    if (sh.overflow != 0 || sh.count > TopShared<THREADS>::kCap) {
      // the lists did not hold: the k-th largest of the slice by counting, which reads it once per bit
      __syncthreads();
      auto each = [&](auto&& f) {
        for (int v = sl.v0 + tid; v < sl.v1; v += THREADS) {
          float e[N];
          Elem<T>::unpack(body[v], e);
#pragma unroll
          for (int i = 0; i < N; ++i) f(rank_code(e[i], sl.head + v * N + i));
        }
        if (edge >= 0) f(edge_code);
      };
      const uint64_t least = block_kth<THREADS>(top, sh.partial, [&](uint64_t t) {
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
    } else if (sh.count > 256) {  // beyond that, ordering by counting costs more
      keep_largest<THREADS>(sh, top);
    }
    found = sh.count;
  }

  // Calls f(place, code) for the `top` largest candidates, places by counting the larger ones.
  auto ordered = [&](auto&& f) {
    if constexpr (TOP) {
      for (int e = tid; e < found; e += THREADS) {
        const uint64_t mine = sh.codes[e];
        int larger = 0;
        for (int i = 0; i < found; ++i) larger += sh.codes[i] > mine ? 1 : 0;
        if (larger < top) f(larger, mine);
      }
    }
  };
  if constexpr (CLUSTER) {
    if (parts > 1) {
      cluster_wait();  // every CTA of the cluster has started
      if constexpr (TOP) {
        if (tid == 0)
          store_cluster_i32(map_to_cta(smem_u32(&joined.merged_count[part]), 0), min(found, top));
        ordered([&](int place, uint64_t code) {
          store_cluster_u64(map_to_cta(smem_u32(&joined.merged[part][place]), 0), code);
        });
      }
      all = cluster_merge<K>(all, c, slots, part, parts);
      if (part != 0) return;
    }
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
  }
  if constexpr (TOP) {
    auto emit = [&](int place, uint64_t code) {
      if (place >= top) return;
      p.top_logprobs[row * top + place] = fmaf(code_value(code) - ref, p.inv_temperature, -log_s);
      p.top_tokens[row * top + place] = (int64_t)code_index(code);
    };
    if (parts == 1) {
      ordered(emit);
    } else if constexpr (CLUSTER) {
      // an entry's place: its place in its own list plus the larger entries of each other list
      for (int e = tid; e < parts * kMaxAlternatives; e += THREADS) {
        const int from = e / kMaxAlternatives, i = e - from * kMaxAlternatives;
        if (i >= joined.merged_count[from]) continue;
        const uint64_t code = joined.merged[from][i];
        int place = i;
        for (int other = 0; other < parts; ++other) {
          if (other == from) continue;
          int lo = 0, hi = joined.merged_count[other];
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (joined.merged[other][mid] > code) lo = mid + 1; else hi = mid;
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
// One bit per logit of the slice marks the listed tokens, a byte per 16-byte vector, so that the sum
// over the others is formed without a subtraction (1 - sum of the listed q would cancel away exactly
// where the student agrees with the teacher).
template <typename T, int THREADS, bool TAIL>
__global__ void __launch_bounds__(THREADS)
distillation_kernel(const RowsView view, const DistillationArgs p) {
  constexpr int N = Elem<T>::kN;
  constexpr int kWarps = THREADS / 32;
  constexpr bool CLUSTER = THREADS == 512;
  constexpr Kind K = TAIL ? kSplit : kSum;
  extern __shared__ __align__(16) uint8_t marks[];
  __shared__ float4 scratch[kWarps];
  __shared__ float4 slots[CLUSTER ? kMaxCluster : 1];
  const int parts = CLUSTER ? p.parts : 1;
  const int part = parts > 1 ? (int)cluster_cta_rank() : 0;
  const int64_t row = parts > 1 ? (int64_t)(blockIdx.x / parts) : (int64_t)blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int vocab = p.vocab;
  const float c = p.inv_temperature * kLog2e;
  const T* x = row_of<T>(view, row);
  const Slice sl = slice_of(x, vocab, part, parts);
  const int64_t* tokens = p.tokens + row * p.top;
  const float* teacher = p.teacher + row * p.top;

  if (!list_counts(p, row)) {  // every warp looks for itself; the row is not read
    if (part == 0 && tid == 0) skip_row(p, row);
    return;
  }
  if (parts > 1) cluster_arrive();
  if (TAIL) {
    const int bytes = sl.v1 - sl.v0;
    for (int i = tid; i < (bytes + 15) / 16; i += THREADS)
      reinterpret_cast<uint4*>(marks)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (warp == 0) {
      for (int k = lane; k < p.top; k += 32) {
        const int64_t token = tokens[k];
        if (token < sl.head || token >= sl.tail_begin) continue;
        const int v = ((int)token - sl.head) / N;
        const int bit = ((int)token - sl.head) - v * N;
        if (v >= sl.v0 && v < sl.v1)
          atomicOr(reinterpret_cast<uint32_t*>(marks) + ((v - sl.v0) >> 2),
                   1u << (8 * ((v - sl.v0) & 3) + bit));
      }
    }
    __syncthreads();
  }
  // the first warp keeps the entries for the end: their logits arrive while the row passes
  int64_t token[kEntriesPerLane];
  float value[kEntriesPerLane], picked[kEntriesPerLane];
#pragma unroll
  for (int i = 0; i < kEntriesPerLane; ++i) {
    const int k = lane + 32 * i;
    token[i] = -1;
    value[i] = -INFINITY;
    picked[i] = __uint_as_float(0x7fffffffu);  // a token outside the vocabulary: NaN
    if (warp == 0 && part == 0 && k < p.top) {
      token[i] = tokens[k];
      if (token[i] >= 0) value[i] = teacher[k];
      if (token[i] >= 0 && token[i] < vocab) picked[i] = Elem<T>::load(x + token[i]);
    }
  }

  // ---- one pass over the logits ----------------------------------------------------------------
  Running run{-INFINITY, 0, 0};
  const int edge = edge_index(sl, vocab, part);
  if (edge >= 0) {
    bool in_list = false;
    if (TAIL)
      for (int k = 0; k < p.top; ++k) in_list |= tokens[k] == edge;
    run = first_of<K>(Elem<T>::load(x + edge), c, in_list);
  }
  const uint4* body = reinterpret_cast<const uint4*>(x + sl.head);
  auto one_sweep = [&](int base, auto full) {
    constexpr bool FULL = decltype(full)::value;
    auto there = [&](int u) { return FULL || base + u * THREADS + tid < sl.v1; };
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (there(u)) raw[u] = body[base + u * THREADS + tid];
    float high = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (there(u)) high = fmaxf(high, Elem<T>::highest(raw[u]));
    if (high > run.m) raise<K>(run, high, c);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (!there(u)) continue;
      float f[N];
      Elem<T>::unpack(raw[u], f);
      accumulate<K>(run, f, c, TAIL ? marks[base + u * THREADS + tid - sl.v0] : 0);
    }
  };
  int base = sl.v0;
  for (; base + THREADS * kUnroll <= sl.v1; base += THREADS * kUnroll)
    one_sweep(base, std::true_type{});
  if (base < sl.v1) one_sweep(base, std::false_type{});
  Stats all = warp_merge<K>(folded(run), c);
  if (lane == 0) scratch[warp] = make_float4(all.m, all.s, all.w, 0.f);
  __syncthreads();
  all = Stats{-INFINITY, 0.f, 0.f};
  if (lane < kWarps) {
    const float4 v = scratch[lane];
    all = Stats{v.x, v.y, v.z};
  }
  all = warp_merge<K>(all, c);
  if constexpr (CLUSTER) {
    if (parts > 1) {
      cluster_wait();  // every CTA of the cluster has started
      all = cluster_merge<K>(all, c, slots, part, parts);
    }
  }
  if (part != 0 || warp != 0) return;

  finish_distillation<TAIL>(p, row, value, picked, reference_of(all.m), TAIL ? all.s + all.w : all.s,
                            all.w);
}

// ---------------------------------------------------------------------------------------------
// Gradients
// ---------------------------------------------------------------------------------------------
// One streaming pass writes the gradient of an unnamed token everywhere (see `GradRow`) and, after a
// barrier, one thread per named token overwrites its element with the full sum (rounded once; a token
// that several entries name is written by the first of them with all their weights, so the order of
// nothing matters).
template <typename T, typename O, int THREADS, bool DISTILL>
__global__ void __launch_bounds__(THREADS)
vocab_grad_kernel(const RowsView view, const VocabGradArgs p) {
  constexpr int N = Elem<T>::kN;
  __shared__ float reduce[THREADS / 32];
  __shared__ int64_t entry_token[kMaxAlternatives + 1];
  __shared__ float entry_weights[kMaxAlternatives + 1];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / p.parts;
  const int part = (int)(blockIdx.x - row * p.parts);
  const int vocab = p.vocab;
  const float c = p.inv_temperature * kLog2e;
  const T* x = row_of<T>(view, row);
  O* out = const_cast<O*>(row_of<O>(p.out, row));
  const Slice sl = slice_of(x, vocab, part, p.parts);
  const int edge = edge_index(sl, vocab, part);

  // ---- the row's coefficients and entries --------------------------------------------------------
  int entries = DISTILL ? p.top : 1;
  float g_top = 0.f;
  bool any_top = false;
  if constexpr (DISTILL) {
    for (int k = tid; k < entries; k += THREADS) {
      entry_token[k] = p.tokens[row * p.top + k];
      entry_weights[k] = entry_token[k] < 0 ? 0.f : entry_weight<true>(p, row, k);
    }
  } else {
    if (tid == 0) {
      entry_token[0] = p.grad != nullptr ? p.tokens[row] : -1;
      entry_weights[0] = entry_weight<false>(p, row, 0);
    }
    if (p.grad_top != nullptr) {
      entries += p.top;
      float mine = 0.f;
      bool any = false;
      for (int k = tid; k < p.top; k += THREADS) {
        const float gk = p.grad_top[row * p.top + k];
        mine += gk;
        any |= gk != 0.f;
        entry_token[1 + k] = p.top_tokens[row * p.top + k];
        entry_weights[1 + k] = gk * p.inv_temperature;
      }
      g_top = block_sum(mine, reduce, THREADS / 32);
      any_top = __syncthreads_or(any) != 0;
    }
  }
  const GradRow g = grad_row<DISTILL>(p, row, g_top, any_top);
  const bool zero = g.zero;

  // ---- every token -----------------------------------------------------------------------------
  auto value = [&](float f, float level) {
    const float t = grad_exponent(f, g.ref, c);
    return fast_exp2(t) * fmaf(g.slope, t, level);
  };
  if (edge >= 0) Elem<O>::store(out + edge, zero ? 0.f : value(Elem<T>::load(x + edge), g.level));
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
        for (int i = 0; i < N; ++i) f[i] = value(f[i], g.level);
      }
      if (aligned) {
        store_vec(out_body + (int64_t)v * N, f);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) Elem<O>::store(out_body + (int64_t)v * N + i, f[i]);
      }
    }
  }
  if (zero) return;

  // ---- the named tokens of this part -----------------------------------------------------------
  __syncthreads();
  for (int k = tid; k < entries; k += THREADS) {
    const int64_t token = entry_token[k];
    bool mine = token >= 0 && token < vocab;
    if (mine) {
      const int64_t in_body = token - sl.head;
      if (token < sl.head || token >= sl.tail_begin)
        mine = part == 0;
      else
        mine = in_body >= (int64_t)sl.v0 * N && in_body < (int64_t)sl.v1 * N;
    }
    for (int j = 0; mine && j < k; ++j) mine = entry_token[j] != token;
    if (mine) {
      float weight = entry_weights[k];
      for (int j = k + 1; j < entries; ++j)
        if (entry_token[j] == token) weight += entry_weights[j];
      Elem<O>::store(out + token, value(Elem<T>::load(x + token), g.level_named) + weight);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------------------------
// CTAs that share a row: as many, up to `most`, as fit the machine at one CTA per SM and leave every
// thread a 16-byte load. A second cluster on an SM costs more than it hides: 64 x 50304 bf16
// log-probabilities take 7.3 us with two CTAs a row, 7.1 with four, 11.3 with eight; one row 6.3 with
// eight against 7.8 with one. Joining top lists costs more with every CTA, hence `most` = 4 there: one
// row with the 20 best 10.4 us with four, 10.5 with one, 12.5 with eight.
int parts_for(int64_t rows, int vocab, int per_vector, int threads, int most) {
  const int vecs = vocab / per_vector;
  int parts = 1;
  while (parts < most && 2 * rows * parts <= device_sm_count() && vecs >= 2 * parts * threads)
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
  a.parts = THREADS == 512 ? parts_for(rows, a.vocab, Elem<T>::kN, THREADS, a.top > 0 ? 4 : kMaxCluster) : 1;
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
  a.parts = THREADS == 512 ? parts_for(rows, a.vocab, N, THREADS, kMaxCluster) : 1;
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

template <typename T, typename O, int THREADS>
void grad_launch(const RowsView& view, VocabGradArgs& a, int64_t rows, bool distill, cudaStream_t stream) {
  const int vecs = a.vocab / Elem<T>::kN;
  a.parts = 1;
  while (a.parts < 64 && rows * a.parts < 8 * device_sm_count() && vecs >= 2 * a.parts * THREADS)
    a.parts *= 2;
  if (distill)
    launch_rows(vocab_grad_kernel<T, O, THREADS, true>, rows * a.parts, 1, THREADS, 0, view, a, stream);
  else
    launch_rows(vocab_grad_kernel<T, O, THREADS, false>, rows * a.parts, 1, THREADS, 0, view, a, stream);
}

// Rows of up to this many bytes have too few vectors for more than 128 threads.
constexpr int64_t kSmallRowBytes = 16 * 1024;

// Gradients of long rows keep 256 threads (8188 x 50304 bf16, distillation: 272 us against 277 with 128;
// 2047 x 50257 fp32 148 against 161), short ones take 128 (16384 x 2048: 62 against 70).
template <typename T, typename O>
void grad_by_shape(const RowsView& view, VocabGradArgs& a, int64_t rows, bool distill, cudaStream_t stream) {
  if ((int64_t)a.vocab * sizeof(T) <= kSmallRowBytes)
    grad_launch<T, O, 128>(view, a, rows, distill, stream);
  else
    grad_launch<T, O, 256>(view, a, rows, distill, stream);
}

// Threads of a CTA, by what there is to hide. Measured on one B200 (50304 bf16 logits a row unless said
// otherwise, log-probabilities / with the 20 best):
//   many rows: small CTAs, of which many share an SM, so that one ends its row (two barriers and a
//     chain of reductions) while others read: 8188 rows 124 / 179 us with 128 threads, 135 / 260 with
//     256, 161 / 395 with 512. Rows of over 128 KB without a top list are long enough for 256: 4096 x
//     131072 161 against 172 us.
//   a few rows per SM: 700 rows 17.4 / 26.8 us with 256, 19.3 / 26.8 with 128.
//   up to two rows per SM: 64 rows 7.3 / 10.5 us with 512, 10.5 / 14.5 with 256, 14.6 / 20.6 with 128;
//     this is also the shape that cuts a row over a cluster.
//   short rows: see kSmallRowBytes.
//   a top list of more than 64 needs more than 128 lanes to take its bound from.
int threads_for(int64_t rows, int64_t row_bytes, int top) {
  const int sms = device_sm_count();
  const bool small = row_bytes <= kSmallRowBytes;
  if (rows <= 2 * sms && !small) return 512;
  if (top > 64) return 256;
  if (rows <= 6 * sms) return small ? 128 : 256;
  return row_bytes <= 128 * 1024 || top > 0 ? 128 : 256;
}

template <typename T>
void logprobs_by_shape(const RowsView& view, TokenLogprobsArgs& a, int64_t rows, cudaStream_t stream) {
  switch (threads_for(rows, (int64_t)a.vocab * sizeof(T), a.top)) {
    case 128: logprobs_launch<T, 128>(view, a, rows, stream); break;
    case 256: logprobs_launch<T, 256>(view, a, rows, stream); break;
    default: logprobs_launch<T, 512>(view, a, rows, stream); break;
  }
}
template <typename T>
void distillation_by_shape(const RowsView& view, DistillationArgs& a, int64_t rows, cudaStream_t stream) {
  switch (threads_for(rows, (int64_t)a.vocab * sizeof(T), 0)) {
    case 128: distillation_launch<T, 128>(view, a, rows, stream); break;
    case 256: distillation_launch<T, 256>(view, a, rows, stream); break;
    default: distillation_launch<T, 512>(view, a, rows, stream); break;
  }
}

}  // namespace

void token_logprobs(const RowsView& view, LogitType type, TokenLogprobsArgs args, int64_t rows,
                    cudaStream_t stream) {
  if (rows == 0) return;
  OB_CHECK(args.top >= 0 && args.top <= kMaxAlternatives && args.top <= args.vocab,
           "token_logprobs: bad number of alternatives");
  switch (type) {
    case LogitType::F32: logprobs_by_shape<float>(view, args, rows, stream); break;
    case LogitType::BF16: logprobs_by_shape<__nv_bfloat16>(view, args, rows, stream); break;
    case LogitType::F16: logprobs_by_shape<__half>(view, args, rows, stream); break;
  }
}

void distillation_loss(const RowsView& view, LogitType type, DistillationArgs args, int64_t rows,
                       cudaStream_t stream) {
  if (rows == 0) return;
  OB_CHECK(args.top >= 1 && args.top <= kMaxAlternatives, "distillation: bad length of the teacher's list");
  switch (type) {
    case LogitType::F32: distillation_by_shape<float>(view, args, rows, stream); break;
    case LogitType::BF16: distillation_by_shape<__nv_bfloat16>(view, args, rows, stream); break;
    case LogitType::F16: distillation_by_shape<__half>(view, args, rows, stream); break;
  }
}

void vocab_grad(const RowsView& view, LogitType type, LogitType out_type, VocabGradArgs args,
                int64_t rows, bool distill, cudaStream_t stream) {
  if (rows == 0) return;
  OB_CHECK(args.top >= 0 && args.top <= kMaxAlternatives, "vocabulary gradient: too many entries");
  if (type == LogitType::F32 && out_type == LogitType::F32)
    grad_by_shape<float, float>(view, args, rows, distill, stream);
  else if (type == LogitType::F32 && out_type == LogitType::BF16)
    grad_by_shape<float, __nv_bfloat16>(view, args, rows, distill, stream);
  else if (type == LogitType::BF16 && out_type == LogitType::BF16)
    grad_by_shape<__nv_bfloat16, __nv_bfloat16>(view, args, rows, distill, stream);
  else if (type == LogitType::F16 && out_type == LogitType::F16)
    grad_by_shape<__half, __half>(view, args, rows, distill, stream);
  else
    OB_CHECK(false, "vocabulary gradient: unsupported types");
}

}  // namespace ob
