// Rows of logits over a vocabulary: log-probabilities of given tokens with
// entropy and the largest alternatives, distillation from a teacher's stored
// logits (a CSR matrix), and both gradients.
//
// With temperature T, c = log2(e) / T, a row's maximum m, u_j = (z_j - m) c,
// e_j = 2^u_j, Z = sum e_j, U = sum e_j u_j:
//   ln q_j  = ln2 (u_j - log2 Z)
//   entropy = ln2 (log2 Z - U / Z)
//   dz_j    = [ g (1[j = token] - q_j) - h q_j (ln q_j + entropy) ] / T
//   loss    = sum_k p_k (ln p_k - ln q_{c_k}),   dz_j = w (q_j - p_j) / T
// A masked place (-inf) has e = 0; a row of nothing else has Z = 0, q = 0.
//
// stats    a workgroup holds a segment of one row in registers: one read gives
//          the maximum, Z, U and, for alternatives, the maxima of groups of
//          elements.
// join     a wave puts a row's segments together and writes the row's results.
//          The k-th largest of the groups' maxima is a lower bound of the k-th
//          largest logit: only the k groups or so that reach it are read again.
// grad     reads a segment again and writes its gradient.
// Long rows of few tokens are split over many workgroups like this, many rows
// fill the chip the same way; the logits' bytes bound all three.  Rows that fit
// the registers of a workgroup take one launch: vocab_rows, distill_rows.
#include "vocab_common.hpp"

using namespace spmm;

namespace {

constexpr int kThreads = 256;
constexpr int kStatsPages = 8, kGradPages = 4;   // pages of 4 KB a workgroup
constexpr int64_t kFill = 256;   // workgroups, before they get more work each
constexpr int kMaxTop = 128;     // alternatives a row
constexpr float kLn2 = 0.693147180559945309f;

// ---- a row ----------------------------------------------------------------------

// A row as 16-byte vectors at aligned addresses (unaligned ones cost a quarter
// of the bandwidth: 820 MB of bf16 rows of odd length 180 us instead of 144),
// with the elements in front of the first and behind the last one, fewer than
// a vector each, as up to 2 N - 2 extra elements.
template <typename T>
struct Row {
  static constexpr int N = Elem<T>::kN;
  const T* z;
  int V, head, nv;   // columns, elements in front of the first vector, vectors
  __device__ __forceinline__ Row(const void* base, int64_t ld, int64_t row, int64_t columns) {
    z = static_cast<const T*>(base) + row * ld;
    V = (int)columns;
    head = (int)((0 - reinterpret_cast<uintptr_t>(z)) & 15) / (int)sizeof(T);
    head = head < V ? head : V;
    nv = (V - head) / N;
  }
  // (past the caches' replacement order, as are the gradients' stores: a step over 4096 x 131072 bf16 502 us
  // instead of 575; at 4 to 128 MB of logits the kernels take between 30 % less and 4 % more)
  __device__ __forceinline__ u32x4 vec(int v) const {
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(z + head + (int64_t)v * N));
  }
  __device__ __forceinline__ int col(int v) const { return head + v * N; }
  // the vector that holds a column, -1: an extra element does
  __device__ __forceinline__ int vec_of(int c) const {
    return c < head || c >= head + nv * N ? -1 : (c - head) / N;
  }
  // column of extra element x of 2 N, or -1
  __device__ __forceinline__ int extra(int x) const {
    const int c = x < N ? (x < head ? x : -1) : head + nv * N + (x - N);
    return x < 2 * N && c < V ? c : -1;
  }
};

// How a row's vectors are split over workgroups: pages of 256 vectors (4 KB),
// VPT of them a workgroup.  Rows of more than VPT pages go to groups of eight
// workgroups that take every eighth page of their span each: what is in flight
// at any time then lies close together (1 GiB copied with 32 KB a workgroup:
// 366 us like this, 402 in one stretch each).  The extra elements belong to the
// first workgroup.
struct Walk {
  int64_t V, S;   // columns, workgroups a row
  int step_log;   // of 1 or 8 (2: the halves of a workgroup of 512 threads)
  __device__ __forceinline__ int page(int seg, int j, int vpt) const {
    return (((seg >> step_log) * vpt + j) << step_log) + (seg & ((1 << step_log) - 1));
  }
  // the workgroup that has a vector (-1: an extra element)
  __device__ __forceinline__ int seg_of(int vec, int vpt) const {
    const int p = vec / 256, in = p & ((1 << step_log) - 1);
    return vec < 0 ? 0 : (((p >> step_log) / vpt) << step_log) + in;
  }
};

// the point that the u_j of a row are measured from
__device__ __forceinline__ float origin(float m) { return m == -kInf ? 0.f : m; }

// (the instruction's results below 2^-126 are zero)
__device__ __forceinline__ float exp2_of(float z, float m, float c) { return __builtin_amdgcn_exp2f((z - m) * c); }
__device__ __forceinline__ float log2_of(float z) { return z == 0.f ? 0.f : __builtin_amdgcn_logf(z); }

struct Part {   // one segment of a row
  float m, z, u, unused;
};

// (value, column) as one number: larger values first, then lower columns; -0 equals +0, NaN is above all
__device__ __forceinline__ uint32_t key_of(float z) {
  if (z != z) return 0xffffffffu;
  const uint32_t b = __float_as_uint(z + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  if (key == 0xffffffffu) return __builtin_nanf("");
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
__device__ __forceinline__ uint64_t entry_of(uint32_t key, int col) {
  return ((uint64_t)key << 32) | (uint32_t)(0x7fffffff - col);
}
__device__ __forceinline__ int col_of(uint64_t entry) { return 0x7fffffff - (int)(uint32_t)entry; }

// ---- statistics -------------------------------------------------------------------

struct StatsArgs {
  const void* z;
  int64_t ld, n;
  Walk wk;
  float c;
  Part* part;
  uint32_t* keys;   // [n * S][256 / lanes] the groups' maxima
  int lanes;        // a group: 1, 2, 4, 8, 16 or 64 neighbouring threads of a workgroup
};

// The statistics of segment t % S of row t / S, by one workgroup (all threads get them).
template <typename T, int VPT, bool ENT, bool TOP>
__device__ __forceinline__ Part segment_stats(const StatsArgs& a, int64_t t, float* red) {
  constexpr int N = Elem<T>::kN;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const Walk wk = a.wk;
  {
    const int64_t row = t / wk.S;
    const int seg = (int)(t - row * wk.S);
    const Row<T> z(a.z, a.ld, row, wk.V);
    u32x4 r[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int first = wk.page(seg, j, VPT) * kThreads;
      if (first >= z.nv) break;   // (uniform)
      r[j] = u32x4{Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf};
      if (first + tid < z.nv) r[j] = z.vec(first + tid);
    }
    const int extra = seg == 0 ? z.extra(tid) : -1;
    const float tail = extra >= 0 ? Elem<T>::load(z.z + extra) : -kInf;
    typename Elem<T>::Max most;
    most.one(tail);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      if (wk.page(seg, j, VPT) * kThreads >= z.nv) break;
      most.vec(r[j]);
    }
    const float mx = most.get(), wm = wave_max(mx);
    if (lane == 0) red[w] = wm;
    __syncthreads();
    const float m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), o = origin(m);
    float zs = 0.f, us = 0.f;
    auto sum = [&](auto masked) {
      zs = us = 0.f;
      auto add = [&](float x) {
        const float u = (x - o) * a.c, e = __builtin_amdgcn_exp2f(u);
        zs += e;
        if (ENT) us = __builtin_fmaf(e, decltype(masked)::value ? fmaxf(u, -1e30f) : u, us);
      };
      if (extra >= 0) add(tail);
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const int first = wk.page(seg, j, VPT) * kThreads;
        if (first >= z.nv) break;
        if (first + tid < z.nv) {
#pragma unroll
          for (int i = 0; i < N; ++i) add(Elem<T>::get(r[j], i));
        }
      }
    };
    sum(std::false_type());
    // 0 times -inf spoils U where places are masked: only such waves keep u finite (one instruction an element)
    if (ENT && __ballot(us != us)) sum(std::true_type());
    const float zw = wave_sum(zs), uw = ENT ? wave_sum(us) : 0.f;
    if (lane == 0) {
      red[4 + w] = zw;
      red[8 + w] = uw;
    }
    __syncthreads();
    const Part part{m, (red[4] + red[5]) + (red[6] + red[7]), (red[8] + red[9]) + (red[10] + red[11]), 0.f};
    if constexpr (TOP) {
      uint32_t key = key_of(mx);
      if (!(zs < kInf)) {   // a NaN among this thread's elements, or +inf
        key = key_of(tail);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
          if (wk.page(seg, j, VPT) * kThreads >= z.nv) break;
#pragma unroll
          for (int i = 0; i < N; ++i) key = max_u(key, key_of(Elem<T>::get(r[j], i)));
        }
      }
      key = a.lanes == 64 ? over_wave(key, max_u) : over_lanes(key, a.lanes, max_u);
      if ((tid & (a.lanes - 1)) == 0) a.keys[t * (kThreads / a.lanes) + tid / a.lanes] = key;
    }
    __syncthreads();   // red is written again
    return part;
  }
}

template <typename T, int VPT, bool TOP>
__global__ __launch_bounds__(kThreads) void vocab_stats(StatsArgs a) {
  __shared__ float red[12];
  for (int64_t t = blockIdx.x; t < a.n * a.wk.S; t += gridDim.x) {
    const Part part = segment_stats<T, VPT, true, TOP>(a, t, red);
    if (threadIdx.x == 0) a.part[t] = part;
  }
}

// A row's segments put together by one wave (all lanes get the result).
struct RowStat {
  float m, z, u;
};
__device__ __forceinline__ RowStat join_parts(const Part* p, int64_t S, float c) {
  const int lane = threadIdx.x & 63;
  float m = -kInf;
  for (int64_t s = lane; s < S; s += 64) m = fmaxf(m, p[s].m);
  m = wave_max(m);
  const float o = origin(m);
  float z = 0.f, u = 0.f;
  for (int64_t s = lane; s < S; s += 64) {
    const Part q = p[s];
    // (a segment of -inf alone has z = 0 unless it holds a NaN)
    const float d = (origin(q.m) - o) * c, f = q.m == -kInf ? 1.f : __builtin_amdgcn_exp2f(d);
    z += q.z * f;
    u += f == 0.f ? 0.f : f * (q.u + (q.m == -kInf ? 0.f : q.z * d));
  }
  z = wave_sum(z);
  return RowStat{m, z < kInf ? z : __builtin_nanf(""), wave_sum(u)};   // (+inf among the logits)
}

// A row in the registers of a workgroup, and its statistics.
template <typename T, int VPT, int THREADS>
struct HeldRow {
  static constexpr int N = Elem<T>::kN, kWaves = THREADS / 64;
  u32x4 r[VPT];
  float tail, mx, zs;   // mx, zs: maximum and sum of this thread's elements
  int extra;
  __device__ __forceinline__ explicit HeldRow(const Row<T>& z) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      r[j] = u32x4{Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf};
      if (j * THREADS + tid < z.nv) r[j] = z.vec(j * THREADS + tid);
    }
    extra = z.extra(tid);
    tail = extra >= 0 ? Elem<T>::load(z.z + extra) : -kInf;
  }
  // red: 3 kWaves floats in LDS, which a barrier behind this call separates from their next use.  ENT: U too
  template <bool ENT>
  __device__ __forceinline__ RowStat stats(const Row<T>& z, float c, float* red) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    typename Elem<T>::Max most;
    most.one(tail);
#pragma unroll
    for (int j = 0; j < VPT; ++j) most.vec(r[j]);
    mx = most.get();
    const float wm = wave_max(mx);
    if (lane == 0) red[w] = wm;
    __syncthreads();
    RowStat st{red[0], 0.f, 0.f};
#pragma unroll
    for (int q = 1; q < kWaves; ++q) st.m = fmaxf(st.m, red[q]);
    const float o = origin(st.m);
    float us = 0.f;
    auto sum = [&](auto masked) {
      zs = us = 0.f;
      auto add = [&](float x) {
        const float u = (x - o) * c, e = __builtin_amdgcn_exp2f(u);
        zs += e;
        if (ENT) us = __builtin_fmaf(e, decltype(masked)::value ? fmaxf(u, -1e30f) : u, us);
      };
      if (extra >= 0) add(tail);
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        if (j * THREADS >= z.nv) break;
        if (j * THREADS + (int)threadIdx.x < z.nv) {
#pragma unroll
          for (int i = 0; i < N; ++i) add(Elem<T>::get(r[j], i));
        }
      }
    };
    sum(std::false_type());
    if (ENT && __ballot(us != us)) sum(std::true_type());   // (0 times -inf, as in segment_stats)
    const float zw = wave_sum(zs), uw = ENT ? wave_sum(us) : 0.f;
    if (lane == 0) {
      red[kWaves + w] = zw;
      red[2 * kWaves + w] = uw;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kWaves; ++q) {
      st.z += red[kWaves + q];
      st.u += red[2 * kWaves + q];
    }
    st.z = st.z < kInf ? st.z : __builtin_nanf("");
    return st;
  }
  // the largest key of this thread's elements, behind stats()
  __device__ __forceinline__ uint32_t key() const {
    uint32_t k = key_of(mx);
    if (!(zs < kInf)) {   // a NaN among them, or +inf
      k = key_of(tail);
#pragma unroll
      for (int j = 0; j < VPT; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) k = max_u(k, key_of(Elem<T>::get(r[j], i)));
    }
    return k;
  }
};

// f(vectors a thread, threads) for rows of up to 32 pages
template <typename F>
void with_rows(int64_t pages, F&& f) {
  if (pages > 16) f(std::integral_constant<int, 8>(), std::integral_constant<int, 1024>());
  else if (pages > 8) f(std::integral_constant<int, 8>(), std::integral_constant<int, 512>());
  else if (pages > 4) f(std::integral_constant<int, 8>(), std::integral_constant<int, 256>());
  else if (pages > 2) f(std::integral_constant<int, 4>(), std::integral_constant<int, 256>());
  else if (pages > 1) f(std::integral_constant<int, 2>(), std::integral_constant<int, 256>());
  else f(std::integral_constant<int, 1>(), std::integral_constant<int, 256>());
}
int64_t pages_of(int64_t V, int type) { return (V / (type == kF32 ? 4 : 8) + kThreads - 1) / kThreads; }

// ---- log-probabilities ------------------------------------------------------------

struct JoinArgs {
  const void* z;
  int64_t ld, n;
  Walk wk;
  int vpt;
  float c, inv_t;
  const Part* part;
  const void* tok;
  int wide, k, lanes;
  const uint32_t* keys;
  float* stat;   // [4][n] log-probability, entropy, maximum, Z
  int64_t* rowptr;
  int32_t* top_col;
  float* top_val;
};

constexpr int kCand = 448;      // candidates of a row that are ranked against each other
constexpr int kHits = 256;      // groups of a row that are read again
constexpr int kKeyRegs = 16;    // groups of a row whose maxima a lane keeps
constexpr int kFlight = 4;      // vectors of a lane that are read at a time

struct TopLds {   // of one wave (four workgroups a CU)
  uint64_t cand[kCand + 8];
  int hit[kHits];
  u32x4 vec[64 * kFlight];   // vectors with a candidate
  int at[64 * kFlight];
};

__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// sum of x over the lanes up to and with this one
__device__ __forceinline__ int wave_scan(int x) {
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

// The k largest logits of a row, in order, to out[0 .. k), by one wave; keys: its
// groups' maxima.
//
// `from`, a key that at least k elements reach, starts as the k-th largest of
// the groups' maxima.  The elements that reach it are collected from the groups
// whose maxima do.  More than kCand: the k-th largest of a sample is a better
// bound, or, if it is the same one, only elements above it are collected, and
// of its equals the lowest columns are looked up in the row.
//
// A wave runs this once, alone on its SIMD or nearly so, and its time goes into
// round trips to memory and into fetching code that no wave has run before: the
// loops are kept short and not unrolled.
template <typename T, typename F>
__device__ __forceinline__ void row_top(const JoinArgs& a, int64_t row, const uint32_t* keys, TopLds& s, F&& out) {
  constexpr int N = Elem<T>::kN;
  const int lane = threadIdx.x & 63, k = a.k;
  const unsigned long long below = (1ull << lane) - 1ull;
  const Row<T> z(a.z, a.ld, row, a.wk.V);
  // vectors a group, and what else is a power of two, as shifts
  const int lanes_log = __builtin_ctz(a.lanes), slots_log = lanes_log + __builtin_ctz(a.vpt), per_log = 8 - lanes_log;
  const int groups = (int)(a.wk.S << per_log);
  const bool in_regs = groups <= 64 * kKeyRegs;
  uint32_t held[kKeyRegs];
#pragma unroll
  for (int j = 0; j < kKeyRegs; ++j) held[j] = in_regs && j * 64 + lane < groups ? keys[j * 64 + lane] : 0u;
  // f(i, key) for all lanes' groups (a lane behind the last has key 0)
  auto each_key = [&](auto&& f) {
    if (in_regs) {
#pragma unroll
      for (int j = 0; j < kKeyRegs; ++j) {
        if (j * 64 >= groups) break;
        f(j * 64 + lane, held[j]);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < groups; i += 64) f(i + lane, i + lane < groups ? keys[i + lane] : 0u);
    }
  };

  // a key that at least k reach, the k-th largest of them unless exactly k do, between lo and hi bit by bit;
  // reach(key): how many are not below it
  auto kth_largest = [&](uint32_t lo, uint32_t hi, auto&& reach) {
    uint32_t key = hi;
    int b = lo == hi ? -1 : 31 - __builtin_clz(lo ^ hi);
    if (b >= 0) key &= ~1u << b;
#pragma unroll 1
    for (; b >= Elem<T>::kLowBits; --b) {
      const uint32_t trial = key | (1u << b);
      const int c = reach(trial);
      if (c >= k) key = trial;
      if (c == k) break;
    }
    // the bits that the type does not have: ones in negative keys and in NaN's
    if (!(key & 0x80000000u) || key > key_of(kInf)) key |= (1u << Elem<T>::kLowBits) - 1u;
    return key;
  };
  // the lanes' largest key, or second largest, is reached by 64 or 128 keys
  uint32_t first = 0, second = 0;
  if (in_regs) {
#pragma unroll
    for (int j = 0; j < kKeyRegs; ++j) {
      const uint32_t low = first < held[j] ? first : held[j];
      second = max_u(second, low);
      first = max_u(first, held[j]);
    }
  }
  const uint32_t least = over_wave(k <= 64 ? first : second, [](uint32_t x, uint32_t y) { return x < y ? x : y; });
  const uint32_t most = in_regs ? over_wave(first, max_u) : ~0u;
  // (64 bits: it may pass the largest key)
  uint64_t from = kth_largest(least, most, [&](uint32_t trial) {
    int c = 0;
    each_key([&](int, uint32_t key) { c += __popcll(__ballot(key >= trial)); });
    return c;
  });
  bool equals = false;   // whether elements of key from - 1 belong to the k largest too
  if (from == key_of(-kInf)) {   // fewer than k groups hold anything else
    ++from;
    equals = true;
  }
  int count;
#pragma unroll 1
  for (;;) {
    int hits = 0;
#pragma unroll 1
    for (;;) {
      hits = 0;
      each_key([&](int i, uint32_t key) {
        const unsigned long long m = __ballot(key >= from);
        if (m == 0) return;
        const int at = hits + __popcll(m & below);
        if (key >= from && at < kHits) s.hit[at] = i;
        hits += __popcll(m);
      });
      if (hits <= kHits) break;
      ++from;   // more than k equal maxima; fewer than k are above them
      equals = true;
    }
    wave_fence();
    count = 0;
    const bool only_nan = from > key_of(kInf);
    const float bound = only_nan ? 0.f : value_of((uint32_t)from);
    auto reaches = [&](float x) { return only_nan ? x != x && from <= 0xffffffffu : !(x < bound); };
    const float may = only_nan ? kInf : bound;   // what reaches `from` is not below it
    auto offer = [&](bool in, float x, int col) {   // (most lanes have nothing)
      const unsigned long long m = __ballot(in && reaches(x));
      if (m == 0) return;
      const int at = count + __popcll(m & below);
      // (of more than kCand a sample of all, so that the next bound leaves a quarter whatever their order)
      const uint32_t slot = at < kCand ? (uint32_t)at : __umulhi((uint32_t)at * 0x9e3779b1u, (uint32_t)at + 1u);
      if (((m >> lane) & 1) && slot < kCand) s.cand[slot] = entry_of(key_of(x), col);
      count += __popcll(m);
    };
    const int vecs = z.nv > 0 ? hits << slots_log : 0;   // (a short row may have extra elements alone)
    auto place = [&](int i) {   // vector i of the hits, or -1
      if (i >= vecs) return -1;
      const int g = s.hit[i >> slots_log], slot = i & ((1 << slots_log) - 1);
      const int thread = ((g << lanes_log) & 255) + (slot & (a.lanes - 1));
      const int v = a.wk.page(g >> per_log, slot >> lanes_log, a.vpt) * kThreads + thread;
      return v < z.nv ? v : -1;
    };
#pragma unroll 1
    for (int i0 = 0; i0 < vecs; i0 += 64 * kFlight) {
      u32x4 x[kFlight];
      int v[kFlight];
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        v[f] = place(i0 + f * 64 + lane);
        x[f] = z.vec(v[f] < 0 ? 0 : v[f]);
      }
      int many = 0;
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        bool any = false;
#pragma unroll
        for (int e = 0; e < N; ++e) any |= !(Elem<T>::get(x[f], e) < may);
        const unsigned long long m = __ballot(any && v[f] >= 0);
        const int at = many + __popcll(m & below);
        if ((m >> lane) & 1) {
          s.vec[at] = x[f];
          s.at[at] = v[f];
        }
        many += __popcll(m);
      }
      wave_fence();
#pragma unroll 1
      for (int i = lane; i - lane < many * N; i += 64) {
        const bool in = i < many * N;
        const int h = in ? i / N : 0;
        offer(in, Elem<T>::load(reinterpret_cast<const T*>(s.vec + h) + i % N), z.col(s.at[h]) + i % N);
      }
      wave_fence();
    }
    {
      const int c = z.extra(lane);
      offer(c >= 0, c >= 0 ? Elem<T>::load(z.z + c) : 0.f, c);
    }
    wave_fence();
    if (count <= kCand) break;
    const uint32_t better = kth_largest(0u, ~0u, [&](uint32_t trial) {
      int c = 0;
#pragma unroll 1
      for (int i = 0; i < kCand; i += 64) c += __popcll(__ballot((uint32_t)(s.cand[i + lane] >> 32) >= trial));
      return c;
    });
    equals = better == from;
    from = equals ? from + 1 : better;
  }
  // of the equals of from - 1 the lowest columns, as many as are missing: the
  // extra elements in front of the vectors, the vectors in order, those behind
  if (equals && count < k) {
    const uint32_t level = (uint32_t)(from - 1);
    const int rounds = (z.nv + 63) / 64;
#pragma unroll 1
    for (int r = -1; r <= rounds && count < k; ++r) {
      const bool vec = r >= 0 && r < rounds && r * 64 + lane < z.nv;
      const int first = r < 0 ? lane : r < rounds ? z.col(r * 64 + lane) : z.col(z.nv) + lane;
      const int elems = vec ? N : (r < 0 ? lane < z.head : r == rounds && first < z.V) ? 1 : 0;
      int many = 0;
      for (int e = 0; e < elems; ++e) many += key_of(Elem<T>::load(z.z + first + e)) == level ? 1 : 0;
      const int incl = wave_scan(many);
      int at = count + incl - many;
      for (int e = 0; e < elems && at < k; ++e)
        if (key_of(Elem<T>::load(z.z + first + e)) == level) s.cand[at++] = entry_of(level, first + e);
      count += __builtin_amdgcn_readlane(incl, 63);
    }
    count = count < k ? count : k;
    wave_fence();
  }
  constexpr int kRead = 8;   // candidates read at a time: the list is filled up with entries below all others
  if (lane < kRead) s.cand[count + lane] = 0;
  wave_fence();
#pragma unroll 1
  for (int i = lane; i < count; i += 64) {
    const uint64_t e = s.cand[i];
    int above = 0;
#pragma unroll 1
    for (int j = 0; j < count; j += kRead) {
      uint64_t o[kRead];
#pragma unroll
      for (int u = 0; u < kRead; ++u) o[u] = s.cand[j + u];
#pragma unroll
      for (int u = 0; u < kRead; ++u) above += o[u] > e ? 1 : 0;
    }
    if (above < k) out(above, e);
  }
  wave_fence();
}

// A row's token: its number and its logit.
struct Token {
  int64_t id;
  float x;
  bool inside;
};
template <typename T>
__device__ __forceinline__ Token token_of(const JoinArgs& a, int64_t row) {
  Token t;
  t.id = token_at(a.tok, a.wide, row);
  t.inside = t.id >= 0 && t.id < a.wk.V;
  t.x = Elem<T>::load(static_cast<const T*>(a.z) + row * a.ld + (t.inside ? t.id : 0));
  return t;
}

// ln q of a row's logit y
__device__ __forceinline__ float ln_q_of(const JoinArgs& a, const RowStat& st, float y) {
  return (y - origin(st.m)) * a.inv_t - kLn2 * log2_of(st.z);
}

// a row's four results, by one thread
__device__ __forceinline__ void write_stat(const JoinArgs& a, int64_t row, const RowStat& st, const Token& t) {
  a.stat[row] = t.inside ? ln_q_of(a, st, t.x) : t.id == -1 ? 0.f : __builtin_nanf("");   // (-1: padding)
  a.stat[a.n + row] = st.z == 0.f ? 0.f : kLn2 * (log2_of(st.z) - st.u / st.z);
  a.stat[2 * a.n + row] = st.m;
  a.stat[3 * a.n + row] = st.z;
}

// a row's alternatives, by one wave
template <typename T>
__device__ __forceinline__ void write_top(const JoinArgs& a, int64_t row, const RowStat& st, const uint32_t* keys,
                                          TopLds& s) {
  if ((threadIdx.x & 63) == 0) {
    a.rowptr[row] = row * a.k;
    if (row == a.n - 1) a.rowptr[a.n] = a.n * a.k;
  }
  row_top<T>(a, row, keys, s, [&](int place, uint64_t e) {
    a.top_col[row * a.k + place] = col_of(e);
    a.top_val[row * a.k + place] = ln_q_of(a, st, value_of((uint32_t)(e >> 32)));
  });
}

// Rows that one workgroup holds: all in one launch.  Its groups are its threads.
template <typename T, int VPT, int THREADS, bool TOP>
__global__ __launch_bounds__(THREADS) void vocab_rows(JoinArgs a) {
  __shared__ float red[THREADS / 64 * 3];
  __shared__ uint32_t keys[TOP ? THREADS : 1];
  __shared__ std::conditional_t<TOP, TopLds, int> top;
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const Token token = token_of<T>(a, row);
    const Row<T> z(a.z, a.ld, row, a.wk.V);
    HeldRow<T, VPT, THREADS> held(z);
    const RowStat st = held.template stats<true>(z, a.c, red);
    if (threadIdx.x == 0) write_stat(a, row, st, token);
    if constexpr (TOP) {
      keys[threadIdx.x] = held.key();
      __syncthreads();
      if (threadIdx.x < 64) write_top<T>(a, row, st, keys, top);
    }
    __syncthreads();
  }
}

// A wave a row.
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void vocab_join(JoinArgs a) {
  __shared__ std::conditional_t<TOP, TopLds, int> top[4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int64_t row = (int64_t)blockIdx.x * 4 + w; row < a.n; row += (int64_t)gridDim.x * 4) {
    const Token token = token_of<T>(a, row);
    const RowStat st = join_parts(a.part + row * a.wk.S, a.wk.S, a.c);
    if (lane == 0) write_stat(a, row, st, token);
    if constexpr (TOP) write_top<T>(a, row, st, a.keys + row * a.wk.S * (kThreads / a.lanes), top[w]);
  }
}

// ---- gradients --------------------------------------------------------------------

// This thread's places of a segment: read at once, written as f(z) later.  An
// output whose rows lie at another alignment than the logits' gets unaligned
// stores.
template <typename T, int VPT>
struct Segment {
  static constexpr int N = Elem<T>::kN;
  u32x4 r[VPT];
  float tail;
  int extra;
  __device__ __forceinline__ Segment(const Row<T>& z, const Walk& wk, int seg) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int v = wk.page(seg, j, VPT) * kThreads + (int)threadIdx.x;
      if (v < z.nv) r[j] = z.vec(v);
    }
    extra = seg == 0 ? z.extra(threadIdx.x) : -1;
    tail = extra >= 0 ? Elem<T>::load(z.z + extra) : 0.f;
  }
  template <typename F>
  __device__ __forceinline__ void write(const Row<T>& z, T* out, const Walk& wk, int seg, F&& f) const {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int v = wk.page(seg, j, VPT) * kThreads + (int)threadIdx.x;
      if (v >= z.nv) break;
      float x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = Elem<T>::get(r[j], i);
      f(x, z.col(v), std::integral_constant<int, N>());
      stream_vec(out + z.col(v), Elem<T>::pack(x));
    }
    if (extra >= 0) {
      float x[1] = {tail};
      f(x, extra, std::integral_constant<int, 1>());
      out[extra] = Elem<T>::cast(x[0]);
    }
  }
};

template <typename T, int VPT>
__device__ __forceinline__ void zero_segment(const Row<T>& z, T* out, const Walk& wk, int seg) {
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int v = wk.page(seg, j, VPT) * kThreads + (int)threadIdx.x;
    if (v < z.nv) stream_vec(out + z.col(v), u32x4{0u, 0u, 0u, 0u});
  }
  const int extra = seg == 0 ? z.extra(threadIdx.x) : -1;
  if (extra >= 0) out[extra] = Elem<T>::cast(0.f);
}

struct TokenGradArgs {
  const void* z;
  int64_t ld, n;
  Walk wk;
  float c, inv_t;
  const void* tok;
  int wide;
  const float *stat, *g, *h;   // g, h: null = 0
  void* out;
  int64_t ldo;
};

// dz_j = e_j (alpha + beta u_j), plus g / T at the token
template <typename T, int VPT, bool ENT>
__global__ __launch_bounds__(kThreads) void vocab_token_grad(TokenGradArgs a) {
  const Walk wk = a.wk;
  const int64_t tasks = a.n * wk.S;
  for (int64_t t = blockIdx.x; t < tasks; t += gridDim.x) {
    const int64_t row = t / wk.S;
    const int seg = (int)(t - row * wk.S);
    const Row<T> z(a.z, a.ld, row, wk.V);
    T* out = static_cast<T*>(a.out) + row * a.ldo;
    const int64_t id = token_at(a.tok, a.wide, row);
    float g = a.g && id != -1 ? a.g[row] * a.inv_t : 0.f;
    const float h = ENT ? a.h[row] * a.inv_t : 0.f;
    if (g == 0.f && h == 0.f) {   // nothing flows into this row: its logits are not read
      zero_segment<T, VPT>(z, out, wk, seg);
      continue;
    }
    const Segment<T, VPT> part(z, wk, seg);
    if (id < -1 || id >= wk.V) g = __builtin_nanf("");
    const float Z = a.stat[3 * a.n + row], l2z = log2_of(Z), rz = Z == 0.f ? 0.f : 1.f / Z;
    const float o = origin(a.stat[2 * a.n + row]);
    const float beta = -h * kLn2 * rz, alpha = -(g + (ENT ? h * (a.stat[a.n + row] - kLn2 * l2z) : 0.f)) * rz;
    part.write(z, out, wk, seg, [&](float* x, int col, auto n) {
      constexpr int n_ = decltype(n)::value;
#pragma unroll
      for (int i = 0; i < n_; ++i) {
        const float u = (x[i] - o) * a.c, e = __builtin_amdgcn_exp2f(u);
        // (e is 0 from -150 down; beta u stays finite for every beta up to 3e34)
        x[i] = ENT ? e * __builtin_fmaf(beta, fmaxf(u, -1e4f), alpha) : e * alpha;
      }
      const int64_t at = id - col;
      if (at >= 0 && at < n_) {
#pragma unroll
        for (int i = 0; i < n_; ++i) x[i] += i == (int)at ? g : 0.f;
      }
    });
  }
}

// ---- distillation -------------------------------------------------------------------

struct Teacher {
  const int64_t* rowptr;
  const int32_t* col;
  const void* val;
  int type;
  int64_t nnz;
  __device__ __forceinline__ float at(int64_t e) const {
    return type == kF32 ? static_cast<const float*>(val)[e]
                        : type == kBF16 ? (float)static_cast<const __bf16*>(val)[e]
                                        : (float)static_cast<const _Float16*>(val)[e];
  }
  // a row's entries, kept inside the arrays whatever the row pointer says
  __device__ __forceinline__ void range(int64_t row, int64_t& b, int64_t& e) const {
    b = rowptr[row];
    e = rowptr[row + 1];
    b = b < 0 ? 0 : (b > nnz ? nnz : b);
    e = e < b ? b : (e > nnz ? nnz : e);
  }
};

struct DistillArgs {
  const void* z;
  int64_t ld, n, V;
  Walk wk;
  float c, inv_t;
  const Part* part;
  int64_t S;            // segments a row in part
  Teacher t;
  float *loss, *stat;   // stat: [n][4] maximum, Z, teacher's maximum and sum
  float* picked;        // [nnz] the student's logits at the teacher's entries
  const float* weight;
  void* out;
  int64_t ldo;
};

// A row of the teacher by one wave: its maximum and sum, and the student's
// logits at its entries, which an output in place of the logits overwrites.
template <typename T>
__device__ __forceinline__ void pick_row(const DistillArgs& a, int64_t row) {
  const int lane = threadIdx.x & 63;
  int64_t b, e;
  a.t.range(row, b, e);
  const T* z = static_cast<const T*>(a.z) + row * a.ld;
  float tm = -kInf;
  bool bad = false;
  for (int64_t i = b + lane; i < e; i += 64) {
    const int32_t col = a.t.col[i];
    bad |= col < -1 || col >= a.V;
    if (col != -1) tm = fmaxf(tm, a.t.at(i));
    if (col >= 0 && col < a.V) a.picked[i] = Elem<T>::load(z + col);
  }
  tm = origin(wave_max(tm));
  bad = __ballot(bad) != 0;
  float ts = 0.f;
  for (int64_t i = b + lane; i < e; i += 64)
    if (a.t.col[i] != -1) ts += exp2_of(a.t.at(i), tm, a.c);
  ts = wave_sum(ts);
  if (lane == 0) {
    a.stat[row * 4 + 2] = tm;
    a.stat[row * 4 + 3] = bad ? __builtin_nanf("") : ts;   // (a column outside the vocabulary)
  }
}

// Statistics of the rows' segments and, in further workgroups, the teacher's.
template <typename T, int VPT>
__global__ __launch_bounds__(kThreads) void distill_stats(StatsArgs s, DistillArgs a) {
  __shared__ float red[12];
  const int64_t segments = a.n * s.wk.S, groups = segments + (a.n + 3) / 4;
  for (int64_t t = blockIdx.x; t < groups; t += gridDim.x) {
    if (t < segments) {
      const Part part = segment_stats<T, VPT, false, false>(s, t, red);
      if (threadIdx.x == 0) s.part[t] = part;
    } else {
      const int64_t row = (t - segments) * 4 + (threadIdx.x >> 6);
      if (row < a.n) pick_row<T>(a, row);
    }
  }
}

// A row's end, by one wave.  loss: the loss and the row's statistics.  With an
// output, what distill_grad left at the teacher's entries of columns that
// own(column) names is replaced by w (q - p) / T, the p of equal columns summed
// in their order, rounded once.
constexpr int kPlaceBits = 13, kRange = 32768;
union FinishLds {   // of one wave
  uint8_t place[1 << kPlaceBits];
  struct {
    uint32_t seen[kRange / 32], twice[kRange / 32];
  } bits;
};

template <typename T, typename F>
__device__ __forceinline__ void finish_row(const DistillArgs& a, int64_t row, FinishLds& s, RowStat st, bool loss,
                                           F&& own) {
  const int lane = threadIdx.x & 63;
  // what does not depend on the row pointer is on its way while that is read
  const float tm = a.stat[row * 4 + 2], ts = a.stat[row * 4 + 3], wt = (a.weight ? a.weight[row] : 1.f) * a.inv_t;
  int64_t b, e;
  a.t.range(row, b, e);
  // a lane's entry of the first 64 (most rows have no more) is read once
  const bool has = b + lane < e;
  const int32_t col0 = has ? a.t.col[b + lane] : -1;
  const float val0 = has ? a.t.at(b + lane) : 0.f, x0 = has ? a.picked[b + lane] : 0.f;
  auto entry = [&](int64_t i, int32_t& col, float& val) {
    const bool first = i == b + lane;
    col = first ? col0 : i < e ? a.t.col[i] : -1;
    val = first ? val0 : i < e ? a.t.at(i) : 0.f;
  };
  const float l2t = log2_of(ts);
  auto share_of = [&](int32_t col, float val) {
    return col != -1 ? __builtin_amdgcn_exp2f((val - tm) * a.c - l2t) : 0.f;
  };
  if (loss) {
    const float o = origin(st.m), l2z = log2_of(st.z);
    float sum = 0.f;
    for (int64_t i = b + lane; i < e; i += 64) {
      int32_t col;
      float val;
      entry(i, col, val);
      if (col < 0 || col >= a.V) continue;
      const float u = (val - tm) * a.c - l2t, p = __builtin_amdgcn_exp2f(u), x = i == b + lane ? x0 : a.picked[i];
      if (!(p == 0.f)) sum += p * (kLn2 * u - ((x - o) * a.inv_t - kLn2 * l2z));
    }
    sum = wave_sum(sum);
    if (ts != ts) sum = st.z = ts;   // a column outside the vocabulary, or a NaN
    if (lane == 0) {
      a.loss[row] = ts == 0.f ? 0.f : sum;   // (no mass: nothing to learn)
      a.stat[row * 4] = st.m;
      a.stat[row * 4 + 1] = st.z;
    }
  }
  if (!a.out || wt == 0.f || ts == 0.f) return;
  const float o = origin(st.m), scale = st.z == 0.f ? 0.f : wt / st.z;
  T* out = static_cast<T*>(a.out) + row * a.ldo;
  auto write = [&](int32_t col, float x, float p) {
    out[col] = Elem<T>::cast(exp2_of(x, o, a.c) * scale - wt * p);
  };
  // the p of the row's entries whose column is a lane's, in order, and whether entry i, that lane's, is the first
  auto search = [&](int64_t i, int32_t mine, float& p, bool& first) {
    p = 0.f;
    for (int64_t from = b; from < e; from += 64) {
      int32_t col;
      float val;
      entry(from + lane, col, val);
      const float share = share_of(col, val);
      const int count = (int)(e - from < 64 ? e - from : 64), before = (int)(i - from < 64 ? i - from : 64);
      for (int j = 0; j < count; ++j) {
        const bool same = (int32_t)__builtin_amdgcn_readlane((uint32_t)col, j) == mine;
        const float share_j = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(share), j));
        p += same ? share_j : 0.f;
        first = first && !(same && j < before);
      }
    }
  };
  if (e - b <= 64) {
    // Equal columns meet in a table: the lane that is left in a place is done, one that finds its own column
    // there has an equal, one that finds another's goes on (two rounds mostly; the search costs 5 us).
    const bool mine = col0 >= 0 && col0 < a.V && own(col0);
    const uint32_t place = ((uint32_t)col0 * 0x9e3779b1u) >> (32 - kPlaceBits);
    bool open = mine, equal = false;
    while (__ballot(open) != 0 && __ballot(equal) == 0) {
      if (open) s.place[place] = (uint8_t)lane;
      wave_fence();
      const int left = open ? (int)s.place[place] : lane;
      wave_fence();
      equal = __shfl(col0, left) == col0 && left != lane;
      open = open && left != lane;
    }
    float p = share_of(col0, val0);
    bool first = mine;
    if (__ballot(equal) != 0) search(b + lane, col0, p, first);
    if (first) write(col0, x0, p);
    return;
  }
  // More entries: a range of columns at a time, in one bit a column, or, where a few entries stand against many
  // ranges, by searching for all of them.
  const int64_t chunks = (e - b + 63) / 64, ranges = (a.V + kRange - 1) / kRange;
  const bool by_range = ranges * (chunks + 3) <= 10 * chunks * chunks;
  for (int64_t r = 0; r < (by_range ? ranges : 1); ++r) {
    const int64_t lo = r * kRange, hi = by_range && lo + kRange < a.V ? lo + kRange : a.V;
    if (by_range) {
      for (int i = lane; i < kRange / 32; i += 64) s.bits.seen[i] = s.bits.twice[i] = 0u;
      wave_fence();
      for (int64_t i = b + lane; i < e; i += 64) {
        const int32_t col = a.t.col[i];
        if (col < lo || col >= hi) continue;
        const int at = (int)(col - lo) >> 5;
        const uint32_t bit = 1u << (col & 31);
        if (atomicOr(&s.bits.seen[at], bit) & bit) atomicOr(&s.bits.twice[at], bit);
      }
      wave_fence();
    }
    for (int64_t base = b; base < e; base += 64) {
      int32_t col;
      float val;
      entry(base + lane, col, val);
      const bool mine = col >= lo && col < hi && own(col);
      const bool equal = !by_range || (mine && ((s.bits.twice[(int)(col - lo) >> 5] >> (col & 31)) & 1));
      float p = share_of(col, val);
      bool first = mine;
      if (__ballot(equal) != 0) search(base + lane, col, p, first);
      if (first) write(col, a.picked[base + lane], p);
    }
    wave_fence();
  }
}

// w q / T in a segment of a row; stat(): the row's statistics, asked for behind
// the loads.  False: nothing flows into the row, which is zero.
template <typename T, int VPT, typename F>
__device__ __forceinline__ bool write_grad(const DistillArgs& a, const Walk& wk, int64_t row, int seg, F&& stat) {
  const Row<T> z(a.z, a.ld, row, wk.V);
  T* out = static_cast<T*>(a.out) + row * a.ldo;
  const float wt = (a.weight ? a.weight[row] : 1.f) * a.inv_t, ts = a.stat[row * 4 + 3];
  if (wt == 0.f || ts == 0.f) {
    zero_segment<T, VPT>(z, out, wk, seg);
    return false;
  }
  const Segment<T, VPT> part(z, wk, seg);
  const RowStat st = stat();
  const float o = origin(st.m), scale = ts != ts ? ts : st.z == 0.f ? 0.f : wt / st.z;
  part.write(z, out, wk, seg, [&](float* x, int, auto n) {
#pragma unroll
    for (int k = 0; k < decltype(n)::value; ++k) x[k] = exp2_of(x[k], o, a.c) * scale;
  });
  return true;
}

// The same everywhere.  JOIN: the rows' statistics are put together here, from
// their segments'.
//
// Bytes bound a step of loss and gradient: the logits are read twice and the
// gradient written once, 3.2 GB for 4096 x 131072 bf16 in 500 us (521 at the
// rate of a large copy).  One read would take a row of 256 KB in registers
// from its statistics to its gradient, half of a CU's: a workgroup a row with
// half of it kept took 574 us, with all of it spilling 670, where these kernels
// then took 580.  A second read out of the last-level cache (statistics and
// gradient of 128 MB at a time) is no faster than one from memory: 660 us.
//
// FINISH: few workgroups, where a launch costs more than it does: each one ends
// its own columns of the row itself, the first one the loss (128 x 131072 bf16
// 21.6 us instead of 22.9 and a launch less for the host, the gradient alone of
// 48 x 32768 fp16 4.3 instead of 5.8; 1000 x 32768, 8000 workgroups, took 52.8
// instead of 47.5).
template <typename T, int VPT, bool JOIN, bool FINISH>
__global__ __launch_bounds__(kThreads) void distill_grad(DistillArgs a) {
  __shared__ std::conditional_t<FINISH, FinishLds, int> lds;
  const Walk wk = a.wk;
  const int64_t tasks = a.n * wk.S;
  for (int64_t t = blockIdx.x; t < tasks; t += gridDim.x) {
    const int64_t row = t / wk.S;
    const int seg = (int)(t - row * wk.S);
    auto stat = [&] {
      return JOIN ? join_parts(a.part + row * a.S, a.S, a.c) : RowStat{a.stat[row * 4], a.stat[row * 4 + 1], 0.f};
    };
    if constexpr (!FINISH) {
      write_grad<T, VPT>(a, wk, row, seg, stat);
    } else {
      RowStat st;
      if (!write_grad<T, VPT>(a, wk, row, seg, [&] { return st = stat(); })) {
        if (!JOIN || seg != 0) continue;   // (the loss is still to be written)
        st = stat();
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // what is replaced has been written
      __syncthreads();
      if (threadIdx.x < 64) {
        const Row<T> z(a.z, a.ld, row, wk.V);
        finish_row<T>(a, row, lds, st, JOIN && seg == 0,
                      [&](int32_t col) { return wk.seg_of(z.vec_of(col), VPT) == seg; });
      }
      __syncthreads();
    }
  }
}

// A wave a row.  LOSS: from the rows' segments, else from their statistics.
template <typename T, bool LOSS>
__global__ __launch_bounds__(kThreads) void distill_finish(DistillArgs a) {
  __shared__ FinishLds lds[kThreads / 64];
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < a.n; row += (int64_t)gridDim.x * 4) {
    const RowStat st = LOSS ? join_parts(a.part + row * a.S, a.S, a.c)
                            : RowStat{a.stat[row * 4], a.stat[row * 4 + 1], 0.f};
    finish_row<T>(a, row, lds[threadIdx.x >> 6], st, LOSS, [](int32_t) { return true; });
  }
}

// Rows that one workgroup holds in registers: loss, statistics and, with an
// output, the gradient in one launch that reads the logits once (GPU time of loss
// and gradient, bf16: 4096 x 32768 113 us instead of 147, 256 x 16000 10.6 instead
// of 14.3, 8000 x 16000 112 instead of 183).  A row's steps wait for each other,
// which costs most where a workgroup fills the CU.
template <typename T, int VPT, int THREADS>
__global__ __launch_bounds__(THREADS) void distill_rows(DistillArgs a) {
  constexpr int N = Elem<T>::kN;
  __shared__ float red[THREADS / 64 * 3];
  __shared__ FinishLds lds;
  const int tid = threadIdx.x, w = tid >> 6;
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const Row<T> z(a.z, a.ld, row, a.V);
    HeldRow<T, VPT, THREADS> held(z);
    if (w == 0) pick_row<T>(a, row);
    const RowStat st = held.template stats<false>(z, a.c, red);
    if (a.out) {
      T* out = static_cast<T*>(a.out) + row * a.ldo;
      const float wt = (a.weight ? a.weight[row] : 1.f) * a.inv_t, ts = a.stat[row * 4 + 3];
      const bool zero = wt == 0.f || ts == 0.f;   // nothing flows into the row
      const float o = origin(st.m), scale = ts != ts ? ts : st.z == 0.f ? 0.f : wt / st.z;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const int v = j * THREADS + tid;
        if (v >= z.nv) break;
        float x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = zero ? 0.f : exp2_of(Elem<T>::get(held.r[j], i), o, a.c) * scale;
        stream_vec(out + z.col(v), Elem<T>::pack(x));
      }
      if (held.extra >= 0) out[held.extra] = Elem<T>::cast(zero ? 0.f : exp2_of(held.tail, o, a.c) * scale);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // what is replaced has been written
      __syncthreads();
    }
    if (w == 0) finish_row<T>(a, row, lds, st, true, [](int32_t) { return true; });
    __syncthreads();
  }
}

// ---- launches -----------------------------------------------------------------------

// Pages a workgroup holds: as many as `most`, fewer in short rows, and fewer
// where the workgroups would not fill the chip.
struct Plan {
  Walk wk;
  int vpt;
};
Plan plan(int64_t n, int64_t V, int type, int most) {
  const int64_t pages = pages_of(V, type);
  Plan p;
  p.vpt = most;
  while (p.vpt > 1 && p.vpt / 2 >= pages) p.vpt /= 2;
  for (;; p.vpt /= 2) {
    const int64_t step = pages > p.vpt ? 8 : 1, span = step * p.vpt, S = (pages + span - 1) / span * step;
    p.wk = Walk{V, S < 1 ? 1 : S, step == 8 ? 3 : 0};
    if (p.vpt == 1 || n * p.wk.S >= kFill) return p;
  }
}
bool sizes_ok(int64_t n, int64_t V, int type) {
  return n >= 0 && V >= 1 && V < (1ll << 31) - 4096 && type >= 0 && type <= 2 && n < (1ll << 40);
}

template <int MOST, typename F>
void with_vpt(int vpt, F&& f) {
  if constexpr (MOST > 1)
    if (vpt < MOST) return with_vpt<MOST / 2>(vpt, f);
  f(std::integral_constant<int, MOST>());
}

// vocab_rows without alternatives: always for rows of up to 16 pages (256 x
// 16000 bf16 4.5 us instead of 7.3, 4096 x 32768 49 instead of 56); a workgroup
// of 16 waves for longer ones fills a CU alone (256 x 65536 9.0 instead of 10.3,
// 1024 35.9 instead of 25.9).  With them it holds its CU while one wave looks for
// them: for few rows (k = 20, 256 x 32768 bf16 12.6 us instead of 17.8, 1024 x
// 8000 11.1 instead of 14.4, 1024 x 16000 19.9 instead of 18.0).
bool in_one_launch(int64_t n, int64_t V, int type, int k) {
  const int64_t pages = pages_of(V, type);
  if (k > 0) return pages <= 16 && n <= 1024 && n * pages <= 4096;
  return pages <= 16 || (pages <= 32 && n <= 256);
}

// The gradient's launches: one where its workgroups are on the chip all at once
constexpr int64_t kFinishGroups = 2048;
template <typename T, bool JOIN>
void launch_grad(const DistillArgs& a, const Plan& q, hipStream_t s) {
  const int64_t groups = a.n * q.wk.S;
  const bool finish = groups <= kFinishGroups;
  with_vpt<kGradPages>(q.vpt, [&](auto e) {
    constexpr int E = decltype(e)::value;
    auto kernel = finish ? distill_grad<T, E, JOIN, true> : distill_grad<T, E, JOIN, false>;
    hipLaunchKernelGGL(kernel, dim3(groups_of(groups)), dim3(kThreads), 0, s, a);
  });
  if (!finish)
    hipLaunchKernelGGL((distill_finish<T, JOIN>), dim3(groups_of((a.n + 3) / 4)), dim3(kThreads), 0, s, a);
}

// distill_rows, or false where the other launches are better: the loss alone has
// no second read to save (1024 rows of 8000 bf16 7.4 us instead of 8.6, 2048 12.9
// instead of 11.9), and a workgroup of 16 waves leaves the chip empty in a short
// call (128 x 65536 bf16 16.4 us instead of 14.8, 256 17.2 instead of 22.3).  So
// does one of 8 waves with few rows: 48 x 32768 fp16 take 11.5 us on the GPU and
// 9.3 in two launches, but a call 14.6 instead of 17.3, as the host bounds it.
template <typename T>
bool launch_rows(const DistillArgs& a, int type, hipStream_t s) {
  const int64_t pages = pages_of(a.V, type);
  if (a.out ? pages > (a.n < 256 ? 16 : 32) : pages > 16 || a.n > 1024) return false;
  with_rows(pages, [&](auto vpt, auto threads) {
    constexpr int kVpt = decltype(vpt)::value, kRowThreads = decltype(threads)::value;
    hipLaunchKernelGGL((distill_rows<T, kVpt, kRowThreads>), dim3(groups_of(a.n)), dim3(kRowThreads), 0, s, a);
  });
  return true;
}

// Threads a group whose maximum is kept for the alternatives: as many as leave
// 16 k groups and 512 in the row, or as few as 1024 groups (a wave's registers)
// allow.  Fewer groups are searched faster, smaller ones are read again faster.
int group_lanes(int64_t S, int k) {
  const int64_t least = 16 * k > 512 ? 16 * k : 512;
  int lanes = 64;
  while (lanes > 1) {
    const int next = lanes == 64 ? 16 : lanes / 2;
    if (S * kThreads / lanes >= least || S * kThreads / next > 64 * kKeyRegs) break;
    lanes = next;
  }
  return lanes;
}

}  // namespace

// bytes of workspace of spmm_token_logprobs (k >= 0) and of the distillation (k = -1)
SPMM_EXPORT int64_t spmm_vocab_ws(int64_t n, int64_t V, int type, int k) {
  if (!sizes_ok(n, V, type) || k < -1 || k > kMaxTop || k > V) return -1;
  if (k >= 0 && in_one_launch(n, V, type, k)) return 0;
  const int64_t S = plan(n, V, type, kStatsPages).wk.S;
  return n * S * (int64_t)(sizeof(Part) + (k > 0 ? kThreads / group_lanes(S, k) * sizeof(uint32_t) : 0));
}

SPMM_EXPORT int spmm_token_logprobs(const void* z, int64_t ld, int64_t n, int64_t V, int type, const void* tok, int wide,
                                    int k, float c, float inv_t, float* stat, int64_t* rowptr, int32_t* top_col,
                                    float* top_val, void* ws, int64_t ws_bytes, hipStream_t s) {
  const int64_t need = spmm_vocab_ws(n, V, type, k);
  if (k < 0 || need < 0 || ws_bytes < need) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  const Plan p = plan(n, V, type, kStatsPages);
  const int64_t S = p.wk.S;
  Part* part = static_cast<Part*>(ws);
  uint32_t* keys = reinterpret_cast<uint32_t*>(part + n * S);
  const int lanes = group_lanes(S, k);
  const StatsArgs sa{z, ld, n, p.wk, c, part, keys, lanes};
  const JoinArgs ja{z, ld, n, p.wk, p.vpt, c, inv_t, part, tok, wide, k, lanes, keys, stat, rowptr, top_col, top_val};
  SPMM_VOCAB_TYPE(type, T, {
    if (in_one_launch(n, V, type, k)) {
      with_rows(pages_of(V, type), [&](auto vpt, auto threads) {
        constexpr int kVpt = decltype(vpt)::value, kRowThreads = decltype(threads)::value;
        JoinArgs ra = ja;
        ra.wk = Walk{V, kRowThreads / kThreads, kRowThreads == 512 ? 1 : 0};
        ra.vpt = kVpt;
        ra.lanes = 1;
        if constexpr (kRowThreads <= 512)
          if (k) {
            hipLaunchKernelGGL((vocab_rows<T, kVpt, kRowThreads, true>), dim3(groups_of(n)), dim3(kRowThreads), 0, s,
                               ra);
            return;
          }
        hipLaunchKernelGGL((vocab_rows<T, kVpt, kRowThreads, false>), dim3(groups_of(n)), dim3(kRowThreads), 0, s, ra);
      });
      SPMM_LAUNCH_CHECK();
      return 0;
    }
    with_vpt<kStatsPages>(p.vpt, [&](auto e) {
      constexpr int E = decltype(e)::value;
      if (k) hipLaunchKernelGGL((vocab_stats<T, E, true>), dim3(groups_of(n * S)), dim3(kThreads), 0, s, sa);
      else hipLaunchKernelGGL((vocab_stats<T, E, false>), dim3(groups_of(n * S)), dim3(kThreads), 0, s, sa);
    });
    SPMM_LAUNCH_CHECK();
    if (k) hipLaunchKernelGGL((vocab_join<T, true>), dim3(groups_of((n + 3) / 4)), dim3(kThreads), 0, s, ja);
    else hipLaunchKernelGGL((vocab_join<T, false>), dim3(groups_of((n + 3) / 4)), dim3(kThreads), 0, s, ja);
    SPMM_LAUNCH_CHECK();
  });
  return 0;
}

SPMM_EXPORT int spmm_token_logprobs_grad(const void* z, int64_t ld, int64_t n, int64_t V, int type, const void* tok,
                                         int wide, float c, float inv_t, const float* stat, const float* g,
                                         const float* h, void* out, int64_t ldo, hipStream_t s) {
  if (!sizes_ok(n, V, type)) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  const Plan p = plan(n, V, type, kGradPages);
  const TokenGradArgs a{z, ld, n, p.wk, c, inv_t, tok, wide, stat, g, h, out, ldo};
  SPMM_VOCAB_TYPE(type, T, {
    with_vpt<kGradPages>(p.vpt, [&](auto e) {
      constexpr int E = decltype(e)::value;
      const dim3 grid(groups_of(n * p.wk.S));
      if (h) hipLaunchKernelGGL((vocab_token_grad<T, E, true>), grid, dim3(kThreads), 0, s, a);
      else hipLaunchKernelGGL((vocab_token_grad<T, E, false>), grid, dim3(kThreads), 0, s, a);
    });
    SPMM_LAUNCH_CHECK();
  });
  return 0;
}

// Loss (and statistics) of every row; with `out` its gradient too.
SPMM_EXPORT int spmm_distill(const void* z, int64_t ld, int64_t n, int64_t V, int type, const int64_t* rowptr,
                             const int32_t* col, const void* val, int val_type, int64_t nnz, float c, float inv_t,
                             float* loss, float* stat, float* picked, const float* weight, void* out, int64_t ldo,
                             void* ws, int64_t ws_bytes, hipStream_t s) {
  const int64_t need = spmm_vocab_ws(n, V, type, -1);
  if (need < 0 || ws_bytes < need || val_type < 0 || val_type > 2) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  const Plan p = plan(n, V, type, kStatsPages), q = plan(n, V, type, kGradPages);
  Part* part = static_cast<Part*>(ws);
  const StatsArgs sa{z, ld, n, p.wk, c, part, nullptr, 1};
  const DistillArgs a{z, ld, n, V, q.wk, c, inv_t, part, p.wk.S, Teacher{rowptr, col, val, val_type, nnz}, loss, stat,
                      picked, weight, out, ldo};
  SPMM_VOCAB_TYPE(type, T, {
    if (launch_rows<T>(a, type, s)) {
      SPMM_LAUNCH_CHECK();
      return 0;
    }
    with_vpt<kStatsPages>(p.vpt, [&](auto e) {
      constexpr int E = decltype(e)::value;
      hipLaunchKernelGGL((distill_stats<T, E>), dim3(groups_of(n * p.wk.S + (n + 3) / 4)), dim3(kThreads), 0, s, sa, a);
    });
    if (out) launch_grad<T, true>(a, q, s);
    else hipLaunchKernelGGL((distill_finish<T, true>), dim3(groups_of((n + 3) / 4)), dim3(kThreads), 0, s, a);
    SPMM_LAUNCH_CHECK();
  });
  return 0;
}

// The gradient alone, from the loss pass's statistics.
SPMM_EXPORT int spmm_distill_grad(const void* z, int64_t ld, int64_t n, int64_t V, int type, const int64_t* rowptr,
                                  const int32_t* col, const void* val, int val_type, int64_t nnz, float c, float inv_t,
                                  const float* stat, const float* picked, const float* weight, void* out, int64_t ldo,
                                  hipStream_t s) {
  if (!sizes_ok(n, V, type) || val_type < 0 || val_type > 2) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  const Plan q = plan(n, V, type, kGradPages);
  const DistillArgs a{z, ld, n, V, q.wk, c, inv_t, nullptr, 0, Teacher{rowptr, col, val, val_type, nnz}, nullptr,
                      const_cast<float*>(stat), const_cast<float*>(picked), weight, out, ldo};
  SPMM_VOCAB_TYPE(type, T, {
    launch_grad<T, false>(a, q, s);
    SPMM_LAUNCH_CHECK();
  });
  return 0;
}
