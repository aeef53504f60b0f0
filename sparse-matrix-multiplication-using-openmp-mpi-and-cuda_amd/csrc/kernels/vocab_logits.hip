// Rows of logits over a vocabulary: log-probabilities of given tokens with
// entropy and the largest alternatives, distillation from a teacher's stored
// logits (a CSR matrix), and both gradients.
//
// With temperature T and c = log2(e) / T, a row's maximum m and u_j = z_j c - m c
// (one fma: the product is not rounded, and what rounding m c costs is the same
// for every j and cancels), e_j = 2^u_j, Z = sum e_j, U = sum e_j u_j:
//   ln q_j  = ln2 (u_j - log2 Z)
//   entropy = ln2 (log2 Z - U / Z)
//   dz_j    = [ g (1[j = token] - q_j) - h q_j (ln q_j + entropy) ] / T
//   loss    = sum_k p_k (ln p_k - ln q_{c_k}),   dz_j = w (q_j - p_j) / T
// A masked place (-inf) has e = 0; a row of nothing else has Z = 0, q = 0.
//
// stats    a workgroup holds a segment of one row in registers: one read gives
//          the maximum, Z, U and the segment's k largest logits.
// join     a wave (a workgroup with alternatives) puts a row's segments together
//          and writes the row's results.
// grad     reads the segment again and writes the gradient.
// Long rows of few tokens are split over many workgroups like this, many rows
// fill the chip the same way; the logits' bytes bound all three.
#include "vocab_common.hpp"

using namespace spmm;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 128;     // alternatives a row
constexpr int kCand = 1024;      // candidates of a segment that are ranked against each other
constexpr float kHuge = 1e37f;   // row maxima whose product with c may overflow
constexpr float kLn2 = 0.693147180559945309f;

struct Part {   // one segment of a row
  float m, z, u, unused;
};

// u_j of a row whose maximum is m
template <bool BIG>
__device__ __forceinline__ float shifted(float z, float m, float mc, float c) {
  return BIG ? (z - m) * c : __builtin_fmaf(z, c, -mc);
}

// the row's maximum as the point that the u_j start from; a row of -inf starts from 0
struct Origin {
  float m, mc;
  bool big;
  __device__ __forceinline__ Origin(float mx, float c) {
#pragma clang fp contract(off)   // m c is rounded, the same everywhere: no use of it may be fused with the product
    m = mx == -kInf ? 0.f : mx;
    mc = m * c;
    big = !(__builtin_fabsf(m) < kHuge);
  }
  __device__ __forceinline__ float at(float z, float c) const {
    return big ? shifted<true>(z, m, mc, c) : shifted<false>(z, m, mc, c);
  }
  // ln q of one logit (natural units throughout where z c might overflow)
  __device__ __forceinline__ float ln_q(float z, float c, float inv_t, float l2z) const {
    if (big || !(__builtin_fabsf(z) < kHuge)) return (z - m) * inv_t - kLn2 * l2z;
    return kLn2 * (shifted<false>(z, m, mc, c) - l2z);
  }
  // how far another origin lies from this one, in the same units
  __device__ __forceinline__ float from(const Origin& o, float c) const {
    return (big || o.big) ? (o.m - m) * c : o.mc - mc;
  }
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

// Sum of one int per thread over the workgroup (all threads get it); scratch: 4 ints.
__device__ __forceinline__ int block_sum(int x, int* scratch) {
  x = wave_sum_i(x);
  __syncthreads();   // earlier reads of scratch are done
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
  __syncthreads();
  return scratch[0] + scratch[1] + scratch[2] + scratch[3];
}

struct TopLds {
  uint64_t cand[kCand];
  float group[kThreads];
  float bound;
  int count;
  int sums[4];
};

// The k largest of the segment's elements, in order, to list[0 .. k).  Each
// thread holds r[VPT] vectors (vector j: columns (v0 + j * 256 + tid) * N ..)
// and one element of the row's tail.  `mine`: the thread's maximum, `odd`:
// whether it holds a NaN.
//
// A k-th largest of the maxima of disjoint groups of elements is a lower bound
// of the k-th largest element, and few elements reach it: those are ranked
// against each other.  Where more than kCand do (equal values, masks) the k-th
// largest key is found bit by bit, and the lowest columns among its equals;
// that reads the segment again, from the caches, and so costs no registers.
template <typename T, int VPT>
__device__ void segment_top(const T* __restrict__ row, const u32x4 (&r)[VPT], int64_t v0, int64_t nv, float tail,
                            int64_t tail_col, bool has_tail, float mine, bool odd, int64_t held, int k,
                            uint64_t* __restrict__ list, TopLds& s) {
  constexpr int N = Elem<T>::kN;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int want = held < k ? (int)held : k;
  for (int i = want + tid; i < k; i += kThreads) list[i] = 0;   // below every entry
  if (want == 0) return;   // (uniform: the segment is empty)
  __syncthreads();
  s.group[tid] = mine;
  if (tid == 0) {
    s.count = 0;
    s.bound = -kInf;
  }
  __syncthreads();
  if (want <= 64) {   // 64 groups: lane l of all four waves
    if (w == 0) {
      const float g = fmaxf(fmaxf(s.group[lane], s.group[64 + lane]), fmaxf(s.group[128 + lane], s.group[192 + lane]));
      int above = 0;
#pragma unroll 8
      for (int j = 0; j < 64; ++j) {
        const float o = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(g), j));
        above += (o > g || (o == g && j < lane)) ? 1 : 0;
      }
      if (above == want - 1) s.bound = g;
    }
  } else if (want <= kThreads) {
    int above = 0;
    for (int j = 0; j < kThreads; ++j) {
      const float o = s.group[j];
      above += (o > mine || (o == mine && j < tid)) ? 1 : 0;
    }
    if (above == want - 1) s.bound = mine;
  }
  __syncthreads();
  const float bound = s.bound;
  auto push = [&](uint32_t key, int col) {
    const int at = atomicAdd(&s.count, 1);
    if (at < kCand) s.cand[at] = entry_of(key, col);
  };
  if (mine >= bound || odd) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int64_t v = v0 + j * kThreads + tid;
      if (v >= nv) break;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float z = Elem<T>::get(r[j], i);
        if (!(z < bound)) push(key_of(z), (int)(v * N + i));
      }
    }
    if (has_tail && !(tail < bound)) push(key_of(tail), (int)tail_col);
  }
  __syncthreads();
  int total = s.count;
  if (total > kCand) {   // (uniform)
    auto each = [&](auto&& f) {   // this thread's elements again
#pragma unroll 1
      for (int j = 0; j < VPT; ++j) {
        const int64_t v = v0 + j * kThreads + tid;
        if (v >= nv) break;
        const u32x4 x = load_vec(row + v * N);
#pragma unroll
        for (int i = 0; i < N; ++i) f(Elem<T>::get(x, i), (int)(v * N + i));
      }
      if (has_tail) f(tail, (int)tail_col);
    };
    uint32_t key = 0;    // the want-th largest key
    for (int b = 31; b >= 0; --b) {
      const uint32_t trial = key | (1u << b);
      int c = 0;
      each([&](float z, int) { c += key_of(z) >= trial ? 1 : 0; });
      if (block_sum(c, s.sums) >= want) key = trial;
    }
    int c = 0;
    each([&](float z, int) { c += key_of(z) > key ? 1 : 0; });
    const int need = want - block_sum(c, s.sums);   // at least one of the equal ones
    int below = 0;                                  // the most columns that hold fewer than `need` of them
    for (int b = 30; b >= 0; --b) {
      const int trial = below | (1 << b);
      c = 0;
      each([&](float z, int col) { c += (key_of(z) == key && col < trial) ? 1 : 0; });
      if (block_sum(c, s.sums) < need) below = trial;
    }
    if (tid == 0) s.count = 0;
    __syncthreads();
    each([&](float z, int col) {
      const uint32_t kz = key_of(z);
      if (kz > key || (kz == key && col <= below)) push(kz, col);
    });
    __syncthreads();
    total = s.count;
  }
  for (int i = tid; i < total; i += kThreads) {
    const uint64_t e = s.cand[i];
    int above = 0;
    for (int j = 0; j < total; ++j) above += s.cand[j] > e ? 1 : 0;
    if (above < want) list[above] = e;
  }
}

struct StatsArgs {
  const void* z;
  int64_t ld, n, V, S;
  float c;
  Part* part;
  int k;
  uint64_t* lists;   // [n * S][k], descending
};

template <typename T, int EPT, bool ENT, bool TOP>
__global__ __launch_bounds__(kThreads) void vocab_stats(StatsArgs a) {
  constexpr int N = Elem<T>::kN, VPT = EPT / N;
  __shared__ float red[12];
  __shared__ std::conditional_t<TOP, TopLds, int> top;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t nv = a.V / N, tasks = a.n * a.S;
  for (int64_t t = blockIdx.x; t < tasks; t += gridDim.x) {
    const int64_t row = t / a.S, seg = t - row * a.S;
    const T* z = static_cast<const T*>(a.z) + row * a.ld;
    const int64_t v0 = seg * kThreads * VPT;
    u32x4 r[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int64_t v = v0 + j * kThreads + tid;
      r[j] = u32x4{Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf};
      if (v < nv) r[j] = load_vec(z + v * N);
    }
    const int64_t tail_col = nv * N + tid;
    const bool has_tail = seg == a.S - 1 && tail_col < a.V;
    const float tail = has_tail ? Elem<T>::load(z + tail_col) : -kInf;
    float mx = tail;
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) mx = fmaxf(mx, Elem<T>::get(r[j], i));
    const float wm = wave_max(mx);
    if (lane == 0) red[w] = wm;
    __syncthreads();
    const float m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const Origin o(m, a.c);
    float zs = 0.f, us = 0.f;
    auto sum = [&](auto big) {
      auto add = [&](float z) {
        const float u = shifted<decltype(big)::value>(z, o.m, o.mc, a.c);
        const float e = __builtin_amdgcn_exp2f(u);
        zs += e;
        if (ENT) us = __builtin_fmaf(e, fmaxf(u, -1e30f), us);   // (0 times -inf)
      };
      add(tail);
#pragma unroll
      for (int j = 0; j < VPT; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) add(Elem<T>::get(r[j], i));
    };
    if (o.big) sum(std::true_type()); else sum(std::false_type());
    const float zw = wave_sum(zs), uw = ENT ? wave_sum(us) : 0.f;
    if (lane == 0) {
      red[4 + w] = zw;
      red[8 + w] = uw;
    }
    __syncthreads();
    if (tid == 0)
      a.part[t] = Part{m, (red[4] + red[5]) + (red[6] + red[7]), (red[8] + red[9]) + (red[10] + red[11]), 0.f};
    if constexpr (TOP) {
      const int64_t left = (nv - v0) * N + (seg == a.S - 1 ? a.V - nv * N : 0);
      const int64_t whole = (int64_t)kThreads * EPT + (seg == a.S - 1 ? a.V - nv * N : 0);
      segment_top<T, VPT>(z, r, v0, nv, tail, tail_col, has_tail, mx, zs != zs, left < whole ? left : whole, a.k,
                          a.lists + t * a.k, top);
    }
    __syncthreads();   // red is written again
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
  const Origin o(m, c);
  float z = 0.f, u = 0.f;
  for (int64_t s = lane; s < S; s += 64) {
    const Part q = p[s];
    const float d = o.from(Origin(q.m, c), c), f = q.m == -kInf ? 1.f : __builtin_amdgcn_exp2f(d);
    // a segment of -inf alone has z = 0, unless it holds a NaN
    z += q.z * f;
    u += f == 0.f ? 0.f : f * (q.u + q.z * (q.m == -kInf ? 0.f : d));
  }
  return RowStat{m, wave_sum(z), wave_sum(u)};
}

struct JoinArgs {
  const void* z;
  int64_t ld, n, V, S;
  float c, inv_t;
  const Part* part;
  const void* tok;
  int wide, k;
  const uint64_t* lists;
  float *logprob, *entropy, *stat;   // stat: [2][n] maximum and Z
  int64_t* rowptr;
  int32_t* top_col;
  float* top_val;
};

constexpr int kMergeLds = 2048;   // entries of a row's lists that are merged in LDS

template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void vocab_join(JoinArgs a) {
  __shared__ uint64_t lds[TOP ? kMergeLds : 1];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t rows = TOP ? a.n : (a.n + 3) / 4;
  for (int64_t t = blockIdx.x; t < rows; t += gridDim.x) {
    const int64_t row = TOP ? t : t * 4 + w;
    if (row >= a.n) return;   // (only without alternatives: no barrier follows)
    const RowStat st = join_parts(a.part + row * a.S, a.S, a.c);
    const Origin o(st.m, a.c);
    const float l2z = st.z == 0.f ? 0.f : __builtin_amdgcn_logf(st.z);
    if (lane == 0 && (!TOP || w == 0)) {
      const int64_t id = token_at(a.tok, a.wide, row);
      float lp = 0.f;   // padding
      if (id >= 0 && id < a.V)
        lp = o.ln_q(Elem<T>::load(static_cast<const T*>(a.z) + row * a.ld + id), a.c, a.inv_t, l2z);
      else if (id != -1)
        lp = __builtin_nanf("");
      a.logprob[row] = lp;
      a.entropy[row] = st.z == 0.f ? 0.f : kLn2 * (l2z - st.u / st.z);
      a.stat[row] = st.m;
      a.stat[a.n + row] = st.z;
    }
    if constexpr (TOP) {
      // every entry's place: how many of the other segments' (descending) lists are above it
      const int k = a.k;
      const int64_t m = a.S * k;
      const uint64_t* all = a.lists + row * m;
      const bool in_lds = m <= kMergeLds;
      __syncthreads();
      if (in_lds)
        for (int64_t i = threadIdx.x; i < m; i += kThreads) lds[i] = all[i];
      __syncthreads();
      const uint64_t* src = in_lds ? lds : all;
      for (int64_t i = threadIdx.x; i < m; i += kThreads) {
        const uint64_t e = src[i];
        if (e == 0) continue;   // a segment shorter than k
        const int64_t own = i / k;
        int place = (int)(i - own * k);
        for (int64_t s = 0; s < a.S && place < k; ++s) {
          if (s == own) continue;
          const uint64_t* l = src + s * k;
          int lo = 0, hi = k;   // entries above e
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (l[mid] > e) lo = mid + 1; else hi = mid;
          }
          place += lo;
        }
        if (place < k) {
          a.top_col[row * k + place] = col_of(e);
          a.top_val[row * k + place] = o.ln_q(value_of((uint32_t)(e >> 32)), a.c, a.inv_t, l2z);
        }
      }
      if (threadIdx.x == 0) {
        a.rowptr[row] = row * k;
        if (row == a.n - 1) a.rowptr[a.n] = a.n * k;
      }
    }
  }
}

struct TokenGradArgs {
  const void* z;
  int64_t ld, n, V, S;
  float c, inv_t;
  const void* tok;
  int wide;
  const float *stat, *entropy, *g, *h;   // g, h: null = 0
  void* out;
  int64_t ldo;
};

// dz_j = e_j (alpha + beta u_j), plus g / T at the token
template <typename T, int EPT, bool ENT>
__global__ __launch_bounds__(kThreads) void vocab_token_grad(TokenGradArgs a) {
  constexpr int N = Elem<T>::kN, VPT = EPT / N;
  const int tid = threadIdx.x;
  const int64_t nv = a.V / N, tasks = a.n * a.S;
  for (int64_t t = blockIdx.x; t < tasks; t += gridDim.x) {
    const int64_t row = t / a.S, seg = t - row * a.S;
    const T* z = static_cast<const T*>(a.z) + row * a.ld;
    T* out = static_cast<T*>(a.out) + row * a.ldo;
    const int64_t v0 = seg * kThreads * VPT, tail_col = nv * N + tid;
    const bool has_tail = seg == a.S - 1 && tail_col < a.V;
    int64_t id = token_at(a.tok, a.wide, row);
    float g = a.g ? a.g[row] * a.inv_t : 0.f;
    const float h = ENT ? a.h[row] * a.inv_t : 0.f;
    if (id == -1) g = 0.f;
    if (g == 0.f && h == 0.f) {   // nothing flows into this row: its logits are not read
      const float zero[N] = {};
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const int64_t v = v0 + j * kThreads + tid;
        if (v < nv) store_vec(out + v * N, Elem<T>::pack(zero));
      }
      if (has_tail) out[tail_col] = Elem<T>::cast(0.f);
      continue;
    }
    if (id < -1 || id >= a.V) g = __builtin_nanf("");
    const float Z = a.stat[a.n + row], l2z = Z == 0.f ? 0.f : __builtin_amdgcn_logf(Z), rz = Z == 0.f ? 0.f : 1.f / Z;
    const Origin o(a.stat[row], a.c);
    const float beta = -h * kLn2 * rz, alpha = -(g + (ENT ? h * (a.entropy[row] - kLn2 * l2z) : 0.f)) * rz;
    u32x4 r[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int64_t v = v0 + j * kThreads + tid;
      if (v < nv) r[j] = load_vec(z + v * N);
    }
    auto write = [&](auto big) {
      auto grad = [&](float x) {
        const float u = shifted<decltype(big)::value>(x, o.m, o.mc, a.c), e = __builtin_amdgcn_exp2f(u);
        return ENT ? e * __builtin_fmaf(beta, fmaxf(u, -1e30f), alpha) : e * alpha;
      };
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const int64_t v = v0 + j * kThreads + tid;
        if (v >= nv) break;
        float x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = grad(Elem<T>::get(r[j], i));
        const int64_t at = id - v * N;
        if (at >= 0 && at < N) {
#pragma unroll
          for (int i = 0; i < N; ++i) x[i] += i == (int)at ? g : 0.f;
        }
        store_vec(out + v * N, Elem<T>::pack(x));
      }
      if (has_tail) out[tail_col] = Elem<T>::cast(grad(Elem<T>::load(z + tail_col)) + (id == tail_col ? g : 0.f));
    };
    if (o.big) write(std::true_type()); else write(std::false_type());
  }
}

// ---- distillation -------------------------------------------------------------
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
  int64_t ld, n, V, S;
  float c, inv_t;
  const Part* part;
  Teacher t;
  float *loss, *stat;   // stat: [n][4] maximum, Z, teacher's maximum and sum
  float* picked;        // [nnz] the student's logits at the teacher's entries
  const float* weight;
  void* out;
  int64_t ldo;
};

// Teacher's statistics and the loss of one row, by one wave.
template <typename T>
__device__ __forceinline__ void distill_row(const DistillArgs& a, int64_t row, RowStat st) {
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
  }
  tm = wave_max(tm);
  const float tm0 = tm == -kInf ? 0.f : tm;
  float ts = 0.f;
  for (int64_t i = b + lane; i < e; i += 64)
    if (a.t.col[i] != -1) ts += __builtin_amdgcn_exp2f((a.t.at(i) - tm0) * a.c);
  ts = wave_sum(ts);
  const Origin o(st.m, a.c);
  const float l2z = st.z == 0.f ? 0.f : __builtin_amdgcn_logf(st.z), l2t = __builtin_amdgcn_logf(ts);
  float loss = 0.f;
  for (int64_t i = b + lane; i < e; i += 64) {
    const int32_t col = a.t.col[i];
    if (col < 0 || col >= a.V) continue;
    const float x = Elem<T>::load(z + col);
    a.picked[i] = x;
    const float u = (a.t.at(i) - tm0) * a.c, p = __builtin_amdgcn_exp2f(u) / ts;
    if (!(p == 0.f)) loss += p * (kLn2 * (u - l2t) - o.ln_q(x, a.c, a.inv_t, l2z));
  }
  loss = wave_sum(loss);
  if (__ballot(bad)) loss = st.z = __builtin_nanf("");   // a column outside the vocabulary
  if (ts == 0.f) loss = __ballot(bad) ? loss : 0.f;      // no mass: nothing to learn
  if (lane == 0) {
    a.loss[row] = loss;
    a.stat[row * 4] = st.m;
    a.stat[row * 4 + 1] = st.z;
    a.stat[row * 4 + 2] = tm0;
    a.stat[row * 4 + 3] = __ballot(bad) ? __builtin_nanf("") : ts;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_join(DistillArgs a) {
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < a.n; row += (int64_t)gridDim.x * 4)
    distill_row<T>(a, row, join_parts(a.part + row * a.S, a.S, a.c));
}

constexpr int kEntries = 1024;   // teacher entries staged in LDS

struct EntryLds {
  int32_t col[kEntries];
  float p[kEntries];
};

// Columns [lo, hi) of a row's gradient where the teacher has entries, written
// over what the dense pass left there: w (q - p) / T with the p of equal
// columns summed in their order, rounded once.  All threads of the workgroup;
// `scale` = w / (T Z), `wt` = w / T.
template <typename T>
__device__ __forceinline__ void distill_entries(const DistillArgs& a, int64_t row, int64_t lo, int64_t hi,
                                                const Origin& o, float scale, float wt, float tm, float ts, T* out,
                                                EntryLds& s) {
  int64_t b, e;
  a.t.range(row, b, e);
  for (int64_t base = b; base < e; base += blockDim.x) {
    const int64_t i = base + threadIdx.x;
    const int32_t mine = i < e ? a.t.col[i] : -1;
    bool first = mine >= lo && mine < hi;
    float p = 0.f;
    for (int64_t from = b; from < e; from += kEntries) {
      const int count = (int)(e - from < kEntries ? e - from : kEntries);
      __syncthreads();
      for (int j = threadIdx.x; j < count; j += blockDim.x) {
        s.col[j] = a.t.col[from + j];
        s.p[j] = __builtin_amdgcn_exp2f((a.t.at(from + j) - tm) * a.c) / ts;
      }
      __syncthreads();
      if (first) {
        for (int j = 0; j < count; ++j) {
          const bool same = s.col[j] == mine;
          first = first && !(same && from + j < i);
          p += same ? s.p[j] : 0.f;
        }
      }
    }
    if (first)
      out[mine] = Elem<T>::cast(__builtin_amdgcn_exp2f(o.at(a.picked[i], a.c)) * scale - wt * p);
  }
}

template <typename T, int EPT>
__global__ __launch_bounds__(kThreads) void distill_grad(DistillArgs a) {
  constexpr int N = Elem<T>::kN, VPT = EPT / N;
  __shared__ EntryLds lds;
  const int tid = threadIdx.x;
  const int64_t nv = a.V / N, tasks = a.n * a.S;
  for (int64_t t = blockIdx.x; t < tasks; t += gridDim.x) {
    const int64_t row = t / a.S, seg = t - row * a.S;
    const T* z = static_cast<const T*>(a.z) + row * a.ld;
    T* out = static_cast<T*>(a.out) + row * a.ldo;
    const int64_t v0 = seg * kThreads * VPT, tail_col = nv * N + tid;
    const bool has_tail = seg == a.S - 1 && tail_col < a.V;
    const float wt = (a.weight ? a.weight[row] : 1.f) * a.inv_t;
    const float Z = a.stat[row * 4 + 1], tm = a.stat[row * 4 + 2], ts = a.stat[row * 4 + 3];
    if (wt == 0.f || ts == 0.f) {   // (uniform) nothing flows into this row
      const float zero[N] = {};
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const int64_t v = v0 + j * kThreads + tid;
        if (v < nv) store_vec(out + v * N, Elem<T>::pack(zero));
      }
      if (has_tail) out[tail_col] = Elem<T>::cast(0.f);
      continue;
    }
    const Origin o(a.stat[row * 4], a.c);
    const float scale = Z == 0.f ? 0.f : wt / Z;
    u32x4 r[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int64_t v = v0 + j * kThreads + tid;
      if (v < nv) r[j] = load_vec(z + v * N);
    }
    auto write = [&](auto big) {
      auto grad = [&](float x) {
        return __builtin_amdgcn_exp2f(shifted<decltype(big)::value>(x, o.m, o.mc, a.c)) * scale;
      };
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const int64_t v = v0 + j * kThreads + tid;
        if (v >= nv) break;
        float x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = grad(Elem<T>::get(r[j], i));
        store_vec(out + v * N, Elem<T>::pack(x));
      }
      if (has_tail) out[tail_col] = Elem<T>::cast(grad(Elem<T>::load(z + tail_col)));
    };
    if (o.big) write(std::true_type()); else write(std::false_type());
    const int64_t lo = v0 * N, whole = lo + (int64_t)kThreads * EPT;
    distill_entries<T>(a, row, lo, seg == a.S - 1 ? a.V : whole, o, scale, wt, tm, ts, out, lds);
    __syncthreads();
  }
}

// ---- launches -------------------------------------------------------------------

// Elements a thread holds.
int elems_of(int64_t V) { return V <= 2048 ? 8 : V <= 4096 ? 16 : V <= 8192 ? 32 : 64; }
int64_t segments(int64_t V, int type, int ept) {
  const int64_t N = type == kF32 ? 4 : 8, nv = V / N, per = (int64_t)kThreads * (ept / N);
  const int64_t s = (nv + per - 1) / per;
  return s < 1 ? 1 : s;
}
bool sizes_ok(int64_t n, int64_t V, int type) {
  return n >= 0 && V >= 1 && V < (1ll << 31) - 4096 && type >= 0 && type <= 2 && n < (1ll << 40);
}

template <typename F>
void with_ept(int ept, F&& f) {
  if (ept == 8) f(std::integral_constant<int, 8>());
  else if (ept == 16) f(std::integral_constant<int, 16>());
  else if (ept == 32) f(std::integral_constant<int, 32>());
  else f(std::integral_constant<int, 64>());
}

}  // namespace

// bytes of workspace of spmm_token_logprobs (k >= 0) and of the distillation (k = 0)
SPMM_EXPORT int64_t spmm_vocab_ws(int64_t n, int64_t V, int type, int k) {
  if (!sizes_ok(n, V, type) || k < 0 || k > kMaxTop || k > V) return -1;
  const int64_t S = segments(V, type, elems_of(V));
  return n * S * (int64_t)(sizeof(Part) + k * sizeof(uint64_t));
}

SPMM_EXPORT int spmm_token_logprobs(const void* z, int64_t ld, int64_t n, int64_t V, int type, const void* tok, int wide,
                                    int k, float c, float inv_t, float* logprob, float* entropy, float* stat, int64_t* rowptr,
                                    int32_t* top_col, float* top_val, void* ws, int64_t ws_bytes, hipStream_t s) {
  const int64_t need = spmm_vocab_ws(n, V, type, k);
  if (need < 0 || ws_bytes < need) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  const int ept = elems_of(V);
  const int64_t S = segments(V, type, ept);
  Part* part = static_cast<Part*>(ws);
  uint64_t* lists = reinterpret_cast<uint64_t*>(part + n * S);
  const StatsArgs sa{z, ld, n, V, S, c, part, k, lists};
  const JoinArgs ja{z, ld, n, V, S, c, inv_t, part, tok, wide, k, lists, logprob, entropy, stat, rowptr, top_col, top_val};
  SPMM_VOCAB_TYPE(type, T, {
    with_ept(ept, [&](auto e) {
      constexpr int E = decltype(e)::value;
      if (k) hipLaunchKernelGGL((vocab_stats<T, E, true, true>), dim3(groups_of(n * S)), dim3(kThreads), 0, s, sa);
      else hipLaunchKernelGGL((vocab_stats<T, E, true, false>), dim3(groups_of(n * S)), dim3(kThreads), 0, s, sa);
    });
    SPMM_LAUNCH_CHECK();
    if (k) hipLaunchKernelGGL((vocab_join<T, true>), dim3(groups_of(n)), dim3(kThreads), 0, s, ja);
    else hipLaunchKernelGGL((vocab_join<T, false>), dim3(groups_of((n + 3) / 4)), dim3(kThreads), 0, s, ja);
    SPMM_LAUNCH_CHECK();
  });
  return 0;
}

SPMM_EXPORT int spmm_token_logprobs_grad(const void* z, int64_t ld, int64_t n, int64_t V, int type, const void* tok,
                                         int wide, float c, float inv_t, const float* stat, const float* entropy,
                                         const float* g, const float* h, void* out, int64_t ldo, hipStream_t s) {
  if (!sizes_ok(n, V, type)) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  const int ept = elems_of(V);
  const int64_t S = segments(V, type, ept);
  const TokenGradArgs a{z, ld, n, V, S, c, inv_t, tok, wide, stat, entropy, g, h, out, ldo};
  SPMM_VOCAB_TYPE(type, T, {
    with_ept(ept, [&](auto e) {
      constexpr int E = decltype(e)::value;
      if (h) hipLaunchKernelGGL((vocab_token_grad<T, E, true>), dim3(groups_of(n * S)), dim3(kThreads), 0, s, a);
      else hipLaunchKernelGGL((vocab_token_grad<T, E, false>), dim3(groups_of(n * S)), dim3(kThreads), 0, s, a);
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
  const int64_t need = spmm_vocab_ws(n, V, type, 0);
  if (need < 0 || ws_bytes < need || val_type < 0 || val_type > 2) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  const int ept = elems_of(V);
  const int64_t S = segments(V, type, ept);
  Part* part = static_cast<Part*>(ws);
  const StatsArgs sa{z, ld, n, V, S, c, part, 0, nullptr};
  const DistillArgs a{z, ld, n, V, S, c, inv_t, part, Teacher{rowptr, col, val, val_type, nnz}, loss, stat, picked,
                      weight, out, ldo};
  SPMM_VOCAB_TYPE(type, T, {
    with_ept(ept, [&](auto e) {
      constexpr int E = decltype(e)::value;
      hipLaunchKernelGGL((vocab_stats<T, E, false, false>), dim3(groups_of(n * S)), dim3(kThreads), 0, s, sa);
      hipLaunchKernelGGL((distill_join<T>), dim3(groups_of((n + 3) / 4)), dim3(kThreads), 0, s, a);
      if (out) hipLaunchKernelGGL((distill_grad<T, E>), dim3(groups_of(n * S)), dim3(kThreads), 0, s, a);
    });
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
  const int ept = elems_of(V);
  const DistillArgs a{z, ld, n, V, segments(V, type, ept), c, inv_t, nullptr, Teacher{rowptr, col, val, val_type, nnz},
                      nullptr, const_cast<float*>(stat), const_cast<float*>(picked), weight, out, ldo};
  SPMM_VOCAB_TYPE(type, T, {
    with_ept(ept, [&](auto e) {
      constexpr int E = decltype(e)::value;
      hipLaunchKernelGGL((distill_grad<T, E>), dim3(groups_of(n * a.S)), dim3(kThreads), 0, s, a);
    });
    SPMM_LAUNCH_CHECK();
  });
  return 0;
}
