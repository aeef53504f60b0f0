// Embedding lookup with scaling, Y = scale * S W, and its gradient by sorted
// tokens, dW = scale * S^T dY, where S is the one-hot CSR matrix of the tokens.
//
// lookup   a group of 8..64 lanes copies one row (or a slice of a long one),
//          16 bytes a lane, four loads in flight.  Bytes bound it: every
//          distinct row read and every output row written once.
// gradient the tokens are sorted with their positions (stable: the sums run
//          over ascending positions, so results are the same in every run),
//          then waves sum tiles of consecutive sorted entries, 16 bytes of
//          columns a lane, and write each token's row when its run ends inside
//          the tile.  A run that crosses tiles leaves fp32 partial rows that a
//          second kernel adds in tile order: a token that fills a tenth of the
//          batch costs the same as any other.  Rows without a token are written
//          as zeros by further workgroups of the same launch.
#include "vocab_common.hpp"

using namespace spmm;

namespace {

// ---- lookup -----------------------------------------------------------------
constexpr int kLookupVecs = 4;   // loads in flight a lane

template <typename T, int LPR>   // LPR lanes a row slice of LPR * kLookupVecs vectors
__global__ __launch_bounds__(256) void embed_lookup(const T* __restrict__ W, int64_t ldw, int64_t V, int64_t D,
                                                    const void* __restrict__ tok, int wide, int64_t n, float scale,
                                                    T* __restrict__ Y, int64_t ldy, int64_t slices) {
  constexpr int N = Elem<T>::kN;
  constexpr int kGroups = 256 / LPR;
  const int lane = threadIdx.x % LPR;
  const int64_t nv = D / N, tasks = n * slices;
  for (int64_t t = (int64_t)blockIdx.x * kGroups + threadIdx.x / LPR; t < tasks; t += (int64_t)gridDim.x * kGroups) {
    const int64_t i = t / slices, s = t - i * slices;
    const int64_t id = token_at(tok, wide, i);
    const bool inside = id >= 0 && id < V;
    const float fill = id == -1 ? 0.f : __builtin_nanf("");   // padding, or a token that the table does not have
    const T* w = W + (inside ? id : 0) * ldw;
    T* y = Y + i * ldy;
    const int64_t v0 = s * LPR * kLookupVecs + lane;
    u32x4 r[kLookupVecs];
    if (inside) {
#pragma unroll
      for (int u = 0; u < kLookupVecs; ++u)
        if (v0 + u * LPR < nv) r[u] = load_vec(w + (v0 + u * LPR) * N);
    }
#pragma unroll
    for (int u = 0; u < kLookupVecs; ++u) {
      if (v0 + u * LPR >= nv) break;
      float x[N];
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = inside ? Elem<T>::get(r[u], e) * scale : fill;
      store_vec(y + (v0 + u * LPR) * N, Elem<T>::pack(x));
    }
    const int64_t c = nv * N + lane;   // the last D % N columns (N <= LPR)
    if (s == slices - 1 && c < D) y[c] = Elem<T>::cast(inside ? Elem<T>::load(w + c) * scale : fill);
  }
}

template <typename T>
int lookup(const T* W, int64_t ldw, int64_t V, int64_t D, const void* tok, int wide, int64_t n, float scale, T* Y,
           int64_t ldy, hipStream_t s) {
  const int64_t nv = D / Elem<T>::kN;
  auto go = [&](auto lpr) {
    constexpr int L = decltype(lpr)::value;
    const int64_t slices = nv > 0 ? (nv + L * kLookupVecs - 1) / (L * kLookupVecs) : 1;
    const int64_t groups = (n * slices + 256 / L - 1) / (256 / L);
    hipLaunchKernelGGL((embed_lookup<T, L>), dim3(groups_of(groups)), dim3(256), 0, s, W, ldw, V, D, tok, wide, n,
                       scale, Y, ldy, slices);
  };
  // the fewest lanes that still hold a row's vectors in one slice
  if (nv <= 8 * kLookupVecs) go(std::integral_constant<int, 8>());
  else if (nv <= 16 * kLookupVecs) go(std::integral_constant<int, 16>());
  else go(std::integral_constant<int, 64>());
  SPMM_LAUNCH_CHECK();
  return 0;
}

// ---- sort of (token, position) ------------------------------------------------
// Keys: the token, or V for padding and for tokens outside the table (sorted
// last, summed nowhere).
__device__ __forceinline__ uint32_t key_of(const void* tok, int wide, int64_t i, int64_t V) {
  const int64_t t = token_at(tok, wide, i);
  return (uint32_t)(t >= 0 && t < V ? t : V);
}

// Few tokens: every token's place is the number of tokens before it, counted
// against all others.  n^2 compares, one launch: at 8192 tokens as long as
// the radix passes' launches, less below.
constexpr int kRankMax = 8192;
constexpr int kRankTile = 2048;

__global__ __launch_bounds__(256) void embed_rank_sort(const void* __restrict__ tok, int wide, int n, int64_t V,
                                                       uint32_t* __restrict__ skey, int32_t* __restrict__ spos) {
  __shared__ uint32_t keys[kRankTile];
  __shared__ int part[4][64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int i = blockIdx.x * 64 + lane;   // the wave's quarter of every tile against the workgroup's 64 tokens
  const uint32_t mine = i < n ? key_of(tok, wide, i, V) : 0u;
  int before = 0;
  for (int base = 0; base < n; base += kRankTile) {
    __syncthreads();
    for (int j = tid; j < kRankTile; j += 256) keys[j] = base + j < n ? key_of(tok, wide, base + j, V) : ~0u;
    __syncthreads();
    const int j0 = w * (kRankTile / 4);
    const int left = n - base - j0, count = left < kRankTile / 4 ? left : kRankTile / 4;
    // equal keys keep their order: those at lower positions count as before
    for (int j = 0; j < count; ++j) {
      const uint32_t k = keys[j0 + j];
      before += (k < mine || (k == mine && base + j0 + j < i)) ? 1 : 0;
    }
  }
  part[w][lane] = before;
  __syncthreads();
  if (w == 0 && i < n) {
    const int at = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
    skey[at] = mine;
    spos[at] = i;
  }
}

// Many tokens: least-significant-digit radix sort, digits of up to 10 bits.
// A wave ranks 16 rounds of 64 keys in order against its own digit counters
// (no workgroup barrier inside), equal digits of a round by ballots.
constexpr int kRounds = 16;
constexpr int kSortTile = 256 * kRounds;   // keys a workgroup
constexpr int kMaxBits = 10;

__global__ __launch_bounds__(256) void embed_digit_count(const void* __restrict__ tok, int wide,
                                                         const uint32_t* __restrict__ key, int64_t n, int64_t V,
                                                         int shift, int bits, int64_t tiles, int32_t* __restrict__ cnt) {
  __shared__ int h[1 << kMaxBits];
  const int bins = 1 << bits;
  for (int b = threadIdx.x; b < bins; b += 256) h[b] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kSortTile;
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = base + r * 256 + threadIdx.x;
    if (i < n) {
      const uint32_t k = key ? key[i] : key_of(tok, wide, i, V);
      atomicAdd(&h[(k >> shift) & (bins - 1)], 1);
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += 256) cnt[(int64_t)b * tiles + blockIdx.x] = h[b];
}

// exclusive scan of the (digit, tile) counters, one workgroup
__global__ __launch_bounds__(1024) void embed_digit_scan(int32_t* __restrict__ cnt, int64_t m) {
  __shared__ int wsum[16];
  __shared__ int carry;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  if (tid == 0) carry = 0;
  for (int64_t base = 0; base < m; base += 1024 * 8) {
    int v[8], s = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t i = base + (int64_t)tid * 8 + u;
      v[u] = i < m ? cnt[i] : 0;
      s += v[u];
    }
    int incl = s;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(incl, d);
      if (lane >= d) incl += y;
    }
    if (lane == 63) wsum[w] = incl;
    __syncthreads();
    int pre = carry, tot = 0;
    for (int q = 0; q < 16; ++q) {
      pre += q < w ? wsum[q] : 0;
      tot += wsum[q];
    }
    int run = pre + incl - s;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t i = base + (int64_t)tid * 8 + u;
      if (i < m) cnt[i] = run;
      run += v[u];
    }
    __syncthreads();   // every read of carry and wsum done
    if (tid == 0) carry += tot;
    __syncthreads();
  }
}

__global__ __launch_bounds__(256) void embed_digit_scatter(const void* __restrict__ tok, int wide,
                                                           const uint32_t* __restrict__ kin,
                                                           const int32_t* __restrict__ pin, int64_t n, int64_t V,
                                                           int shift, int bits, int64_t tiles,
                                                           const int32_t* __restrict__ offs, uint32_t* __restrict__ kout,
                                                           int32_t* __restrict__ pout) {
  __shared__ int wcnt[4][1 << kMaxBits];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, bins = 1 << bits;
  for (int b = tid; b < bins; b += 256) wcnt[0][b] = wcnt[1][b] = wcnt[2][b] = wcnt[3][b] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kSortTile + (int64_t)w * (64 * kRounds);
  const unsigned long long below = (1ull << lane) - 1ull;
  uint32_t k[kRounds];
  int rank[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = base + r * 64 + lane;
    k[r] = i < n ? (kin ? kin[i] : key_of(tok, wide, i, V)) : 0u;
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const bool ok = base + r * 64 + lane < n;
    const int d = (int)(k[r] >> shift) & (bins - 1);
    unsigned long long m = __ballot(ok);
    for (int b = 0; b < bits; ++b) {
      const unsigned long long bb = __ballot((d >> b) & 1);
      m &= ((d >> b) & 1) ? bb : ~bb;
    }
    const int in_round = __popcll(m & below);
    // (one wave, whose LDS accesses stay in order: every lane reads a round's counter before the
    // digit's first lane raises it, and the next round reads what that lane wrote)
    const int seen = ok ? wcnt[w][d] : 0;
    rank[r] = seen + in_round;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (ok && in_round == 0) wcnt[w][d] = seen + __popcll(m);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = base + r * 64 + lane;
    if (i >= n) continue;
    const int d = (int)(k[r] >> shift) & (bins - 1);
    int at = offs[(int64_t)d * tiles + blockIdx.x] + rank[r];
    for (int q = 0; q < w; ++q) at += wcnt[q][d];
    kout[at] = k[r];
    pout[at] = pin ? pin[i] : (int32_t)i;
  }
}

// ---- sums ---------------------------------------------------------------------
struct GradArgs {
  const void* dy;
  int64_t lddy;
  const uint32_t* skey;
  const int32_t* spos;
  int64_t n, V, D, ldw, tiles, slices, vblocks;
  float scale;
  void* dw;
  float* part;   // [tiles][2][D]: a tile's sums of the run it begins inside and of the one it ends inside
  int accumulate;
};

constexpr int kTile = 32;       // sorted entries a wave
constexpr int kFlight = 8;      // row loads in flight
constexpr int kFillRows = 16;   // table rows a zero-filling wave

// N floats of columns [c, c + N) (fewer at the row's end), from / to a row of any of the types
template <typename T, int N>
__device__ __forceinline__ void load_cols(const T* row, int64_t c, int64_t D, float (&x)[N]) {
  if (c + N <= D) {
#pragma unroll
    for (int b = 0; b < N; b += Elem<T>::kN) {
      const u32x4 r = load_vec(row + c + b);
#pragma unroll
      for (int e = 0; e < Elem<T>::kN; ++e) x[b + e] = Elem<T>::get(r, e);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = c + e < D ? Elem<T>::load(row + c + e) : 0.f;
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_cols(T* row, int64_t c, int64_t D, const float (&x)[N]) {
  if (c + N <= D) {
#pragma unroll
    for (int b = 0; b < N; b += Elem<T>::kN) store_vec(row + c + b, Elem<T>::pack(x + b));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c + e < D) row[c + e] = Elem<T>::cast(x[e]);
  }
}

// the finished fp32 sum of one token's row: scaled, added to what is there, rounded once
template <typename TO, int N>
__device__ __forceinline__ void finish_row(const GradArgs& a, int64_t v, int64_t c, float (&acc)[N]) {
  TO* row = static_cast<TO*>(a.dw) + v * a.ldw;
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] *= a.scale;
  if (a.accumulate) {
    float old[N];
    load_cols<TO, N>(row, c, a.D, old);
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] += old[e];
  }
  store_cols<TO, N>(row, c, a.D, acc);
}

template <typename TI, typename TO>
__global__ __launch_bounds__(256) void embed_grad_sum(GradArgs a) {
  constexpr int N = Elem<TI>::kN;
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), waves = (int64_t)gridDim.x * 4;
  const int64_t sums = a.tiles * a.slices, tasks = sums + a.vblocks;
  for (int64_t t = wave; t < tasks; t += waves) {
    if (t >= sums) {   // zero rows for tokens that the batch does not have
      const int64_t v0 = (t - sums) * kFillRows;
      // lane r finds where row v0 + r would start among the sorted keys
      int64_t lo = 0, hi = a.n;
      const int64_t v = v0 + (lane < kFillRows ? lane : kFillRows - 1);
      while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if ((int64_t)a.skey[mid] < v) lo = mid + 1; else hi = mid;
      }
      const bool empty = v < a.V && (lo >= a.n || (int64_t)a.skey[lo] != v);
      const unsigned long long m = __ballot(empty);
      constexpr int NO = Elem<TO>::kN;
      const float zero[NO] = {};
      for (int r = 0; r < kFillRows; ++r) {
        if (!((m >> r) & 1)) continue;
        TO* row = static_cast<TO*>(a.dw) + (v0 + r) * a.ldw;
        for (int64_t c = (int64_t)lane * NO; c < a.D; c += 64 * NO) store_cols<TO, NO>(row, c, a.D, zero);
      }
      continue;
    }
    const int64_t tile = t / a.slices, c = ((t - tile * a.slices) * 64 + lane) * N;
    const int64_t b = tile * kTile, e = b + kTile < a.n ? b + kTile : a.n;
    const bool mine = c < a.D;
    // the tile's tokens and positions, one a lane (a padded lane repeats the last)
    const int64_t at = b + lane < e ? b + lane : e - 1;
    const int key = (int)a.skey[at], pos = a.spos[at];
    const int V = (int)a.V;
    const int before = b > 0 ? (int)a.skey[b - 1] : -1, after = e < a.n ? (int)a.skey[e] : -1;
    const int cnt = (int)(e - b);
    float acc[N] = {};
    bool head = true;   // the current run reaches back to the tile's first entry
    for (int r0 = 0; r0 < cnt; r0 += kFlight) {
      float x[kFlight][N];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        const int r = r0 + u < cnt ? r0 + u : cnt - 1;
        const int64_t p = __builtin_amdgcn_readlane(pos, r);
        if (mine && __builtin_amdgcn_readlane(key, r) < V)
          load_cols<TI, N>(static_cast<const TI*>(a.dy) + p * a.lddy, c, a.D, x[u]);
      }
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        const int r = r0 + u;
        if (r >= cnt) break;
        const int kr = __builtin_amdgcn_readlane(key, r);
        if (kr >= V) break;   // padding: nothing behind it either
        const int next = r + 1 < cnt ? __builtin_amdgcn_readlane(key, r + 1) : after;
#pragma unroll
        for (int q = 0; q < N; ++q) acc[q] += x[u][q];
        if (next == kr && r + 1 < cnt) continue;
        const bool from_before = head && before == kr, into_next = r + 1 == cnt && after == kr;
        if (mine) {
          if (!from_before && !into_next) {
            finish_row<TO, N>(a, kr, c, acc);
          } else {   // slot 0: a run that began in an earlier tile; slot 1: one that goes on from here
            float* p = a.part + (tile * 2 + (from_before ? 0 : 1)) * a.D;
            store_cols<float, N>(p, c, a.D, acc);
          }
        }
#pragma unroll
        for (int q = 0; q < N; ++q) acc[q] = 0.f;
        head = false;
      }
    }
  }
}

// Runs that cross tiles: the tile where a run begins adds its own partial row
// and those of the tiles that the run goes through, in order.  Four waves take
// a quarter of the tiles each.
template <typename TI, typename TO>
__global__ __launch_bounds__(256) void embed_grad_join(GradArgs a) {
  constexpr int N = 4;   // columns a lane: partial rows are fp32
  __shared__ float sums[3][64 * N];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t slices = (a.D + 64 * N - 1) / (64 * N), tasks = a.tiles * slices;
  for (int64_t t = blockIdx.x; t < tasks; t += gridDim.x) {
    const int64_t tile = t / slices, c = ((t - tile * slices) * 64 + lane) * N;
    const int64_t b = tile * kTile, e = b + kTile;
    if (e >= a.n) continue;   // (uniform) nothing follows the last tile
    const uint32_t key = a.skey[e - 1];
    if (key >= (uint32_t)a.V || a.skey[e] != key) continue;          // no run crosses here
    if (a.skey[b] == key && b > 0 && a.skey[b - 1] == key) continue; // it began in an earlier tile
    // the last tile that the run reaches
    int64_t lo = e, hi = a.n;   // first entry behind the run
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (a.skey[mid] <= key) lo = mid + 1; else hi = mid;
    }
    const int64_t last = (lo - 1) / kTile, m = last - tile + 1;   // partial rows: this tile's and those behind it
    const int64_t q0 = m * w / 4, q1 = m * (w + 1) / 4;
    float acc[N] = {};
    for (int64_t q = q0; q < q1; q += kFlight) {
      float x[kFlight][N];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        const int64_t i = q + u < q1 ? q + u : q1 - 1;
        if (c < a.D) load_cols<float, N>(a.part + ((tile + i) * 2 + (i == 0 ? 1 : 0)) * a.D, c, a.D, x[u]);
      }
#pragma unroll
      for (int u = 0; u < kFlight; ++u)
        if (q + u < q1) {
#pragma unroll
          for (int s = 0; s < N; ++s) acc[s] += x[u][s];
        }
    }
    __syncthreads();
    if (w > 0) {
#pragma unroll
      for (int s = 0; s < N; ++s) sums[w - 1][lane * N + s] = acc[s];
    }
    __syncthreads();
    if (w == 0 && c < a.D) {
#pragma unroll
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int s = 0; s < N; ++s) acc[s] += sums[q][lane * N + s];
      if constexpr (Elem<TO>::kN == N) {
        finish_row<TO, N>(a, key, c, acc);
      } else {   // 16-bit outputs: four columns are half a vector
        TO* row = static_cast<TO*>(a.dw) + (int64_t)key * a.ldw;
#pragma unroll
        for (int s = 0; s < N; ++s) {
          if (c + s >= a.D) break;
          float x = acc[s] * a.scale;
          if (a.accumulate) x += Elem<TO>::load(row + c + s);
          row[c + s] = Elem<TO>::cast(x);
        }
      }
    }
  }
}

struct GradSizes {
  int64_t tiles, sort_tiles, keys, part, cnt, total;
  int bits, passes;
};

// Layout of the workspace: sorted keys and positions (twice for the radix
// passes), digit counters, partial rows.
bool grad_sizes(int64_t n, int64_t V, int64_t D, GradSizes& g) {
  if (n < 0 || n >= (1ll << 31) - kSortTile || V < 1 || V >= (1ll << 31) - 1 || D < 1) return false;
  int total_bits = 1;
  while ((V >> total_bits) != 0) ++total_bits;   // keys 0 .. V
  g.passes = (total_bits + kMaxBits - 1) / kMaxBits;
  g.bits = (total_bits + g.passes - 1) / g.passes;
  g.tiles = (n + kTile - 1) / kTile;
  g.sort_tiles = (n + kSortTile - 1) / kSortTile;
  g.keys = (n + 63) / 64 * 64;
  g.cnt = n > kRankMax ? ((int64_t)g.sort_tiles << g.bits) : 0;
  g.part = g.tiles * 2 * D;
  const int64_t copies = n > kRankMax ? 2 : 1;
  g.total = (g.keys * 2 * copies + (g.cnt + 63) / 64 * 64) * 4 + g.part * 4;
  return true;
}

template <typename TI, typename TO>
int grad(GradArgs a, hipStream_t s) {
  const int64_t waves = a.tiles * a.slices + a.vblocks;
  if (waves > 0)
    hipLaunchKernelGGL((embed_grad_sum<TI, TO>), dim3(groups_of((waves + 3) / 4)), dim3(256), 0, s, a);
  SPMM_LAUNCH_CHECK();
  if (a.tiles > 1) {
    const int64_t joins = a.tiles * ((a.D + 255) / 256);
    hipLaunchKernelGGL((embed_grad_join<TI, TO>), dim3(groups_of(joins)), dim3(256), 0, s, a);
    SPMM_LAUNCH_CHECK();
  }
  return 0;
}

}  // namespace

SPMM_EXPORT int spmm_embedding(const void* W, int64_t ldw, int64_t V, int64_t D, int type, const void* tok, int wide,
                               int64_t n, float scale, void* Y, int64_t ldy, hipStream_t s) {
  if (n < 0 || V < 0 || D < 0) return (int)hipErrorInvalidValue;
  if (n == 0 || D == 0) return 0;
  SPMM_VOCAB_TYPE(type, T,
                  return lookup<T>(static_cast<const T*>(W), ldw, V, D, tok, wide, n, scale, static_cast<T*>(Y), ldy, s));
  return 0;
}

// bytes of workspace, or -1 for sizes that the kernels do not take
SPMM_EXPORT int64_t spmm_embedding_grad_ws(int64_t n, int64_t V, int64_t D) {
  GradSizes g;
  return grad_sizes(n, V, D, g) ? g.total : -1;
}

SPMM_EXPORT int spmm_embedding_grad(const void* dy, int64_t lddy, int in_type, const void* tok, int wide, int64_t n,
                                    int64_t V, int64_t D, float scale, void* dw, int64_t ldw, int out_type,
                                    int accumulate, void* ws, int64_t ws_bytes, hipStream_t s) {
  GradSizes g;
  if (!grad_sizes(n, V, D, g) || ws_bytes < g.total) return (int)hipErrorInvalidValue;
  uint32_t* ka = static_cast<uint32_t*>(ws);
  int32_t* pa = reinterpret_cast<int32_t*>(ka + g.keys);
  uint32_t* skey = ka;
  int32_t* spos = pa;
  char* behind = reinterpret_cast<char*>(pa + g.keys);
  if (n > kRankMax) {
    uint32_t* kb = reinterpret_cast<uint32_t*>(behind);
    int32_t* pb = reinterpret_cast<int32_t*>(kb + g.keys);
    int32_t* cnt = pb + g.keys;
    behind = reinterpret_cast<char*>(cnt + (g.cnt + 63) / 64 * 64);
    const uint32_t* kin = nullptr;
    const int32_t* pin = nullptr;
    uint32_t* kout = ka;
    int32_t* pout = pa;
    for (int p = 0; p < g.passes; ++p) {
      const int shift = p * g.bits;
      hipLaunchKernelGGL(embed_digit_count, dim3((unsigned)g.sort_tiles), dim3(256), 0, s, tok, wide, kin, n, V, shift,
                         g.bits, g.sort_tiles, cnt);
      hipLaunchKernelGGL(embed_digit_scan, dim3(1), dim3(1024), 0, s, cnt, g.cnt);
      hipLaunchKernelGGL(embed_digit_scatter, dim3((unsigned)g.sort_tiles), dim3(256), 0, s, tok, wide, kin, pin, n, V,
                         shift, g.bits, g.sort_tiles, cnt, kout, pout);
      kin = kout;
      pin = pout;
      kout = kout == ka ? kb : ka;
      pout = pout == pa ? pb : pa;
    }
    skey = const_cast<uint32_t*>(kin);
    spos = const_cast<int32_t*>(pin);
  } else if (n > 0) {
    hipLaunchKernelGGL(embed_rank_sort, dim3((unsigned)((n + 63) / 64)), dim3(256), 0, s, tok, wide, (int)n, V, skey,
                       spos);
  }
  SPMM_LAUNCH_CHECK();
  GradArgs a;
  a.dy = dy;
  a.lddy = lddy;
  a.skey = skey;
  a.spos = spos;
  a.n = n;
  a.V = V;
  a.D = D;
  a.ldw = ldw;
  a.tiles = g.tiles;
  a.vblocks = accumulate ? 0 : (V + kFillRows - 1) / kFillRows;
  a.scale = scale;
  a.dw = dw;
  a.part = reinterpret_cast<float*>(behind);
  a.accumulate = accumulate;
  SPMM_VOCAB_TYPE(in_type, TI, {
    a.slices = (D + 64 * Elem<TI>::kN - 1) / (64 * Elem<TI>::kN);
    if (out_type == kF32) return grad<TI, float>(a, s);
    if (out_type == in_type) return grad<TI, TI>(a, s);
    return (int)hipErrorInvalidValue;
  });
  return 0;
}
