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
//          as zeros by further workgroups of the same launch, or of the sort's.
//          A short batch is not sorted at all (embed_grad_brief).
#include "vocab_common.hpp"

using namespace spmm;

namespace {

// ---- lookup -----------------------------------------------------------------
constexpr int kLookupVecs = 4;   // loads in flight a lane

// LPR lanes a row slice of LPR * kLookupVecs vectors.  STREAM: an output of over
// 16 MB leaves the table's rows in the caches (32768 x 4096 bf16: 65 us instead of 77).
template <typename T, int LPR, bool STREAM>
__global__ __launch_bounds__(256) void embed_lookup(const T* __restrict__ W, int64_t ldw, int64_t V, int64_t D,
                                                    const void* __restrict__ tok, int wide, int64_t n, float scale,
                                                    T* __restrict__ Y, int64_t ldy, int64_t slices) {
  constexpr int N = Elem<T>::kN;
  constexpr int kGroups = 256 / LPR;
  const int lane = threadIdx.x % LPR;
  const int64_t nv = D / N, tasks = n * slices;
  for (int64_t t = (int64_t)blockIdx.x * kGroups + threadIdx.x / LPR; t < tasks; t += (int64_t)gridDim.x * kGroups) {
    // (a 64-bit division costs as much as the copy of a short row)
    const int64_t i = tasks <= 0xffffffffll ? (int64_t)((uint32_t)t / (uint32_t)slices) : t / slices;
    const int64_t s = t - i * slices;
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
      T* to = y + (v0 + u * LPR) * N;
      if (STREAM) stream_vec(to, Elem<T>::pack(x)); else store_vec(to, Elem<T>::pack(x));
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
    const bool stream = n * D * (int64_t)sizeof(T) >= kStreamBytes;
    auto kernel = stream ? embed_lookup<T, L, true> : embed_lookup<T, L, false>;
    hipLaunchKernelGGL(kernel, dim3(groups_of(groups)), dim3(256), 0, s, W, ldw, V, D, tok, wide, n, scale, Y, ldy,
                       slices);
  };
  // the fewest lanes that still hold a row's vectors in one slice
  if (nv <= 8 * kLookupVecs) go(std::integral_constant<int, 8>());
  else if (nv <= 16 * kLookupVecs) go(std::integral_constant<int, 16>());
  else go(std::integral_constant<int, 64>());
  SPMM_LAUNCH_CHECK();
  return 0;
}

// `bytes` zeros from thread `first` of `threads` on: vectors, then the last columns
__device__ __forceinline__ void zero_table(uint16_t* table, int64_t bytes, int64_t first, int64_t threads) {
  const int64_t vecs = bytes / 16;
  for (int64_t i = first; i < vecs; i += threads) store_vec(table + i * 8, u32x4{0u, 0u, 0u, 0u});
  if (first < (bytes & 15) / 2) table[vecs * 8 + first] = 0;
}

__global__ __launch_bounds__(256) void embed_zero(uint16_t* __restrict__ table, int64_t bytes) {
  zero_table(table, bytes, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}

// ---- sort of (token, position) ------------------------------------------------
// Keys: the token, or V for padding and for tokens outside the table (sorted
// last, summed nowhere).  The last pass also writes slot[token], one of the
// token's places among the sorted keys: a row v has a token if slot[v] is a
// place and the key there is v, whatever slot[v] held before, so that nothing
// has to be cleared.
__device__ __forceinline__ uint32_t key_of(const void* tok, int wide, int64_t i, int64_t V) {
  const int64_t t = token_at(tok, wide, i);
  return (uint32_t)(t >= 0 && t < V ? t : V);
}

// Few tokens: every token's place is the number of tokens before it, counted
// against all others by the 16 waves of a workgroup for its 64 tokens.  One
// launch and n^2 compares: 5 us at 777 tokens, 15 at 8192, 25 at 16384, where
// the radix passes' four launches take 22.
constexpr int kRankMax = 12288;
constexpr int kRankTile = 4096;   // keys in LDS
constexpr int kRankWaves = 16;

// A table of which the batch has few rows, without gaps between them, is zeroed
// by further workgroups of this launch (`bytes` of it), before any row is
// known: the sort hides behind that.  8000 tokens over 65536 x 4096 bf16: 120 us
// instead of 133, 12000 over 131072 x 513: 55 instead of 63.
constexpr int64_t kFewRows = 8;   // table rows for each token, from which on

__global__ __launch_bounds__(64 * kRankWaves) void embed_rank_sort(const void* __restrict__ tok, int wide, int n,
                                                                   int64_t V, uint32_t* __restrict__ skey,
                                                                   int32_t* __restrict__ spos,
                                                                   int32_t* __restrict__ slot,
                                                                   uint16_t* __restrict__ table, int64_t bytes) {
  __shared__ __attribute__((aligned(16))) uint32_t keys[kRankTile];
  __shared__ int part[kRankWaves][64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, sorts = (n + 63) / 64;
  if ((int)blockIdx.x >= sorts) {
    zero_table(table, bytes, (int64_t)(blockIdx.x - sorts) * (64 * kRankWaves) + tid,
               (int64_t)(gridDim.x - sorts) * (64 * kRankWaves));
    return;
  }
  const int i = blockIdx.x * 64 + lane;
  const uint32_t mine = i < n ? key_of(tok, wide, i, V) : 0u;
  int before = 0;
  for (int base = 0; base < n; base += kRankTile) {
    const int held = n - base < kRankTile ? n - base : kRankTile, blocks = (held + 63) / 64;
    __syncthreads();
    for (int j = tid; j < blocks * 64; j += 64 * kRankWaves) keys[j] = j < held ? key_of(tok, wide, base + j, V) : ~0u;
    __syncthreads();
    for (int b = w; b < blocks; b += kRankWaves) {
      const u32x4* k4 = reinterpret_cast<const u32x4*>(keys + b * 64);
      const int own = (int)blockIdx.x - base / 64;   // the workgroup's own tokens are that block
      // equal keys keep their order: those of earlier blocks are before, of later ones behind
      if (b < own) {
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const u32x4 k = k4[q];
          before += (k[0] <= mine) + (k[1] <= mine) + (k[2] <= mine) + (k[3] <= mine);
        }
      } else if (b > own) {
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const u32x4 k = k4[q];
          before += (k[0] < mine) + (k[1] < mine) + (k[2] < mine) + (k[3] < mine);
        }
      } else {
#pragma unroll 4
        for (int q = 0; q < 64; ++q) {
          const uint32_t k = keys[b * 64 + q];
          before += (k < mine || (k == mine && q < lane)) ? 1 : 0;
        }
      }
    }
  }
  part[w][lane] = before;
  __syncthreads();
  if (w == 0 && i < n) {
    int at = 0;
#pragma unroll
    for (int q = 0; q < kRankWaves; ++q) at += part[q][lane];
    skey[at] = mine;
    spos[at] = i;
    if (slot && mine < (uint32_t)V) slot[mine] = at;
  }
}

// Many tokens: least-significant-digit radix sort, digits of up to 10 bits.
// A wave ranks its rounds of 64 keys in order against its own digit counters
// (no workgroup barrier inside), equal digits of a round by ballots.  With few
// tiles every scatter workgroup adds up the counters in front of it by itself;
// with many a scan of its own does it once.
constexpr int kMaxBits = 10;
constexpr int kSmallRounds = 4, kLargeRounds = 16;   // keys a wave / 64
constexpr int64_t kFewTiles = 128;

__global__ __launch_bounds__(256) void embed_digit_count(const void* __restrict__ tok, int wide,
                                                         const uint32_t* __restrict__ key, int64_t n, int64_t V,
                                                         int shift, int bits, int rounds, int32_t* __restrict__ cnt) {
  __shared__ int h[1 << kMaxBits];
  const int bins = 1 << bits;
  for (int b = threadIdx.x; b < bins; b += 256) h[b] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * 256 * rounds;
#pragma unroll 4
  for (int r = 0; r < rounds; ++r) {
    const int64_t i = base + r * 256 + threadIdx.x;
    if (i < n) {
      const uint32_t k = key ? key[i] : key_of(tok, wide, i, V);
      atomicAdd(&h[(k >> shift) & (bins - 1)], 1);
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += 256) cnt[((int64_t)blockIdx.x << bits) + b] = h[b];
}

// Where each digit of a tile starts among all keys, from the tiles' counters
// [tile][digit]: keys of smaller digits, then those of this digit in the tiles
// in front.  One workgroup of 256 threads; start[] in LDS.
template <int PER>   // consecutive digits a thread
__device__ __forceinline__ void digit_starts(const int32_t* __restrict__ cnt, int64_t tiles, int64_t tile, int bits,
                                             int* start, int* wsum) {
  constexpr int kLoads = 16;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, bins = 1 << bits;
  const int first = tid * PER < bins ? tid * PER : 0;
  int front[PER] = {}, total[PER] = {};
  for (int64_t t0 = 0; t0 < tiles; t0 += kLoads) {
    int c[kLoads][PER];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int64_t t = t0 + u < tiles ? t0 + u : tiles - 1;
#pragma unroll
      for (int q = 0; q < PER; ++q) c[u][q] = cnt[(t << bits) + first + q];
    }
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        const int x = t0 + u < tiles ? c[u][q] : 0;
        total[q] += x;
        front[q] += t0 + u < tile ? x : 0;
      }
  }
  int s = 0;
#pragma unroll
  for (int q = 0; q < PER; ++q) s += tid * PER < bins ? total[q] : 0;
  int incl = s;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(incl, d);
    if (lane >= d) incl += y;
  }
  if (lane == 63) wsum[w] = incl;
  __syncthreads();
  int run = incl - s;
  for (int q = 0; q < w; ++q) run += wsum[q];
  if (tid * PER < bins) {
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      start[tid * PER + q] = run + front[q];
      run += total[q];
    }
  }
}

// The same for many tiles, once a pass: cnt becomes the starts.  Digit by
// digit over the tiles, then over the digits' totals; one workgroup.
__global__ __launch_bounds__(1024) void embed_digit_scan(int32_t* __restrict__ cnt, int64_t tiles, int bits) {
  __shared__ int wsum[16];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, bins = 1 << bits;
  int total = 0;
  if (tid < bins)
    for (int64_t t0 = 0; t0 < tiles; t0 += 16) {
      int c[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) c[u] = t0 + u < tiles ? cnt[((t0 + u) << bits) + tid] : 0;
#pragma unroll
      for (int u = 0; u < 16; ++u) total += c[u];
    }
  int incl = total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(incl, d);
    if (lane >= d) incl += y;
  }
  if (lane == 63) wsum[w] = incl;
  __syncthreads();
  int run = incl - total;
  for (int q = 0; q < w; ++q) run += wsum[q];
  if (tid < bins)
    for (int64_t t0 = 0; t0 < tiles; t0 += 16) {
      int c[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) c[u] = t0 + u < tiles ? cnt[((t0 + u) << bits) + tid] : 0;
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        if (t0 + u < tiles) cnt[((t0 + u) << bits) + tid] = run;
        run += c[u];
      }
    }
}

template <int R>
__global__ __launch_bounds__(256) void embed_digit_scatter(const void* __restrict__ tok, int wide,
                                                           const uint32_t* __restrict__ kin,
                                                           const int32_t* __restrict__ pin, int64_t n, int64_t V,
                                                           int shift, int bits, int64_t tiles, int scanned,
                                                           const int32_t* __restrict__ cnt, uint32_t* __restrict__ kout,
                                                           int32_t* __restrict__ pout, int32_t* __restrict__ slot) {
  __shared__ int wcnt[4][1 << kMaxBits];
  __shared__ int start[1 << kMaxBits];
  __shared__ int wsum[4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, bins = 1 << bits;
  for (int b = tid; b < bins; b += 256) wcnt[0][b] = wcnt[1][b] = wcnt[2][b] = wcnt[3][b] = 0;
  const int64_t base = (int64_t)blockIdx.x * (256 * R) + (int64_t)w * (64 * R);
  const unsigned long long below = (1ull << lane) - 1ull;
  uint32_t k[R];
  int32_t pos[R];
  int rank[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t i = base + r * 64 + lane;
    k[r] = i < n ? (kin ? kin[i] : key_of(tok, wide, i, V)) : 0u;
    pos[r] = i < n ? (pin ? pin[i] : (int32_t)i) : 0;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
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
  if (scanned) {
    for (int b = tid; b < bins; b += 256) start[b] = cnt[((int64_t)blockIdx.x << bits) + b];
  } else {
    if (bits <= 8) digit_starts<1>(cnt, tiles, blockIdx.x, bits, start, wsum);
    else if (bits == 9) digit_starts<2>(cnt, tiles, blockIdx.x, bits, start, wsum);
    else digit_starts<4>(cnt, tiles, blockIdx.x, bits, start, wsum);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (base + r * 64 + lane >= n) continue;
    const int d = (int)(k[r] >> shift) & (bins - 1);
    int at = start[d] + rank[r];
    for (int q = 0; q < w; ++q) at += wcnt[q][d];
    kout[at] = k[r];
    pout[at] = pos[r];
    if (slot && k[r] < (uint32_t)V) slot[k[r]] = at;
  }
}

// ---- sums ---------------------------------------------------------------------
// tile: sorted entries a wave of embed_grad_sum; fill: table rows a workgroup looks through for
// empty ones, 0: parts of long rows; fills: such workgroups
struct GradArgs {
  const void* dy;
  int64_t lddy;
  const uint32_t* skey;
  const int32_t *spos, *slot;
  int64_t n, V, D, ldw, tile, tiles, slices, fill, fills;
  float scale;
  void* dw;
  float* part;   // [tiles][2][D]: a tile's sums of the run it begins inside and of the one it ends inside
  int accumulate, zeroed;   // rows without a token: they keep their values; they are zero already
  int brief;                // embed_grad_brief, without sorted entries
};

// Sorted entries a wave sums.  A wave hides its loads behind those of other
// waves, so it gets few entries where the chip's 1024 SIMDs would have few waves
// otherwise: up to 6144 tokens times slices waves of 8 are at most 768, up to
// 65536 waves of 16 at most 4096, and above that waves of 32 at least 2048.  The
// whole gradient of mixed tokens with 8, 16 and 32 entries a wave: 3000 of 500
// columns 25, 31 and 41 us; 32000 of 256 47, 45 and 48; 20548 of 857 54, 55 and
// 59; 12000 of 4096 90, 82 and 79; 65536 of 1024 110, 98 and 90.  A token that
// fills much of the batch asks for more, as one workgroup a slice joins its
// partial rows: half of the 32000 117, 80 and 66 us, all of them 199, 118 and 80.
inline int64_t tile_of(int64_t entries) {   // tokens times slices
  return entries <= 6144 ? 8 : entries <= 65536 ? 16 : 32;
}
constexpr int kFlight = 8;   // row loads in flight
constexpr int64_t kNarrow = 8;   // columns, below which rows are summed by embed_grad_narrow
constexpr int kFillBytes = 16384, kFillPieces = 8;

// The first of the sorted keys at or behind lo that is not before v: 64 probes a step.
__device__ __forceinline__ int64_t first_not_before(const uint32_t* __restrict__ skey, int64_t lo, int64_t n, int64_t v) {
  const int lane = threadIdx.x & 63;
  int64_t hi = n;
  while (lo < hi) {
    const int64_t step = (hi - lo + 63) / 64, i = lo + lane * step;
    const int c = __popcll(__ballot(i < hi && (int64_t)skey[i] < v));   // the probes before v are the first ones
    if (c == 0) return lo;
    const int64_t end = lo + c * step;
    lo += (c - 1) * step + 1;
    hi = end < hi ? end : hi;
  }
  return lo;
}

// Columns [c, c + N) of a row of any of the types.  A row's last lane reaches
// back (`from` = D - N < c) so that every lane reads whole vectors; what it
// reads of its neighbour's columns is summed and not written.
template <typename T, int N>
struct Cols {
  static constexpr int kVecs = N / Elem<T>::kN > 0 ? N / Elem<T>::kN : 1;
  u32x4 v[kVecs];
  __device__ __forceinline__ void load(const T* row, int64_t from) {
#pragma unroll
    for (int b = 0; b < kVecs; ++b) v[b] = load_vec(row + from + b * Elem<T>::kN);
  }
  __device__ __forceinline__ void fetch(const T* row, int64_t from) {   // what is read once
#pragma unroll
    for (int b = 0; b < kVecs; ++b) v[b] = fetch_vec(row + from + b * Elem<T>::kN);
  }
  __device__ __forceinline__ float get(int e) const { return Elem<T>::get(v[e / Elem<T>::kN], e % Elem<T>::kN); }
};

template <typename T, int N>
__device__ __forceinline__ void store_cols(T* row, int64_t c, int64_t from, const float (&x)[N]) {
  if (from == c) {
#pragma unroll
    for (int b = 0; b < N; b += Elem<T>::kN) store_vec(row + c + b, Elem<T>::pack(x + b));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (from + e >= c) row[from + e] = Elem<T>::cast(x[e]);
  }
}

// the finished fp32 sum of one token's row: scaled, added to what is there, rounded once
template <typename TO, int N>
__device__ __forceinline__ void finish_row(const GradArgs& a, int64_t v, int64_t c, int64_t from, float (&acc)[N]) {
  TO* row = static_cast<TO*>(a.dw) + v * a.ldw;
  if (a.accumulate) {
    Cols<TO, N> old;
    old.load(row, from);
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = __builtin_fmaf(acc[e], a.scale, old.get(e));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] *= a.scale;
  }
  store_cols<TO, N>(row, c, from, acc);
}

__device__ __forceinline__ bool row_is_empty(const GradArgs& a, int64_t v) {
  const uint32_t at = (uint32_t)a.slot[v];
  return !((int64_t)at < a.n && (int64_t)a.skey[at] == v);
}

// Zero rows for tokens that the batch does not have, as pieces of 4 KB of a
// long row or as groups of short rows.  Eight consecutive workgroups write
// every eighth piece of their span each, so that the writes in flight lie close
// together: 1 GiB of such writes takes 166 us, of 32 or 64 KB a workgroup in
// one stretch 189 and 197.  One piece a workgroup (157) would look for its row
// each time, which costs more than it gives (470 us).
template <typename TO>
__device__ __forceinline__ void fill_piece(const GradArgs& a, int64_t piece) {
  constexpr int NO = Elem<TO>::kN;
  const int lane = threadIdx.x & 63;
  const unsigned nv = (unsigned)(a.D / NO), tail = (unsigned)(a.D % NO);
  if (a.fill == 0) {
    const int64_t per = (nv + 255) / 256, pieces = a.V * per;
    const int64_t base = (piece / 8) * 8 * kFillPieces + piece % 8;
    if (base >= pieces) return;
    const int64_t mine = base + 8 * lane;   // lane j looks for the row of piece j
    const unsigned long long empty = __ballot(lane < kFillPieces && mine < pieces && row_is_empty(a, mine / per));
#pragma unroll
    for (int j = 0; j < kFillPieces; ++j) {
      if (!((empty >> j) & 1)) continue;
      const int64_t p = base + 8 * j, r = p / per;
      const unsigned i = (unsigned)(p - r * per) * 256 + threadIdx.x;
      TO* row = static_cast<TO*>(a.dw) + r * a.ldw;
      if (i < nv) store_vec(row + (int64_t)i * NO, u32x4{0u, 0u, 0u, 0u});
      if (p - r * per == per - 1 && threadIdx.x < tail) row[(int64_t)nv * NO + threadIdx.x] = Elem<TO>::cast(0.f);
    }
    return;
  }
  const int64_t v0 = piece * a.fill;
  const int rows = (int)(a.V - v0 < a.fill ? a.V - v0 : a.fill);
  const unsigned long long empty = __ballot(lane < rows && row_is_empty(a, v0 + lane));
  TO* first = static_cast<TO*>(a.dw) + v0 * a.ldw;
  for (unsigned i = threadIdx.x; i < rows * nv; i += 256) {
    const unsigned r = i / nv;
    if ((empty >> r) & 1) store_vec(first + (int64_t)r * a.ldw + (int64_t)(i - r * nv) * NO, u32x4{0u, 0u, 0u, 0u});
  }
  for (unsigned i = threadIdx.x; i < rows * tail; i += 256) {
    const unsigned r = i / tail;
    if ((empty >> r) & 1) first[(int64_t)r * a.ldw + (int64_t)nv * NO + (i - r * tail)] = Elem<TO>::cast(0.f);
  }
}

template <typename TI, typename TO>
__global__ __launch_bounds__(256) void embed_grad_sum(GradArgs a) {
  constexpr int N = Elem<TI>::kN;
  const int lane = threadIdx.x & 63;
  const int64_t sums = a.tiles * a.slices, sum_groups = (sums + 3) / 4;
  for (int64_t group = blockIdx.x; group < sum_groups + a.fills; group += gridDim.x) {
    if (group >= sum_groups) {
      fill_piece<TO>(a, group - sum_groups);
      continue;
    }
    const int64_t t = group * 4 + (threadIdx.x >> 6);
    if (t >= sums) continue;
    const int64_t tile = t / a.slices, c = ((t - tile * a.slices) * 64 + lane) * N;
    const int64_t b = tile * a.tile, e = b + a.tile < a.n ? b + a.tile : a.n;
    const bool mine = c < a.D;
    const int64_t from = c + N <= a.D ? c : a.D - N;   // (D >= N)
    // the tile's tokens and positions, one a lane (further lanes repeat the last)
    const int64_t at = b + lane < e ? b + lane : e - 1;
    const int key = (int)a.skey[at], pos = a.spos[at];
    const int V = (int)a.V;
    const int before = b > 0 ? (int)a.skey[b - 1] : -1, after = e < a.n ? (int)a.skey[e] : -1;
    const int cnt = (int)(e - b);
    float acc[N] = {};
    bool head = true;   // the current run reaches back to the tile's first entry
    for (int r0 = 0; r0 < cnt && __builtin_amdgcn_readlane(key, r0) < V; r0 += kFlight) {
      Cols<TI, N> x[kFlight];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {   // (behind the last entry: that one again)
        const int64_t i = __builtin_amdgcn_readlane(pos, r0 + u < cnt ? r0 + u : cnt - 1);
        x[u].fetch(static_cast<const TI*>(a.dy) + i * a.lddy, from);
      }
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        const int r = r0 + u;
        if (r >= cnt) break;
        const int kr = __builtin_amdgcn_readlane(key, r);
        if (kr >= V) break;   // padding: nothing behind it either
        const int next = r + 1 < cnt ? __builtin_amdgcn_readlane(key, r + 1) : after;
#pragma unroll
        for (int q = 0; q < N; ++q) acc[q] += x[u].get(q);
        if (next == kr && r + 1 < cnt) continue;
        const bool from_before = head && before == kr, into_next = r + 1 == cnt && after == kr;
        if (mine) {
          if (!from_before && !into_next) {
            finish_row<TO, N>(a, kr, c, from, acc);
          } else {   // slot 0: a run that began in an earlier tile; slot 1: one that goes on from here
            store_cols<float, N>(a.part + (tile * 2 + (from_before ? 0 : 1)) * a.D, c, from, acc);
          }
        }
#pragma unroll
        for (int q = 0; q < N; ++q) acc[q] = 0.f;
        head = false;
      }
    }
  }
}

// Rows narrower than a vector (of the 16-bit types): a wave a table row, whose lanes take every 64th
// of its sorted entries (200000 tokens over 50000 rows of 4 fp32: 98 us; all of
// them one token: 2.0 ms).
template <typename TI, typename TO>
__global__ __launch_bounds__(256) void embed_grad_narrow(GradArgs a) {
  constexpr int kMost = (int)kNarrow - 1;
  const int lane = threadIdx.x & 63, D = (int)a.D;
  for (int64_t v = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); v < a.V; v += (int64_t)gridDim.x * 4) {
    const int64_t first = first_not_before(a.skey, 0, a.n, v);
    const bool any = first < a.n && (int64_t)a.skey[first] == v;
    if (a.accumulate && !any) continue;
    float acc[kMost] = {};
    const int64_t end = any ? first_not_before(a.skey, first, a.n, v + 1) : first;
#pragma unroll 4
    for (int64_t i = first + lane; i < end; i += 64) {
      const TI* x = static_cast<const TI*>(a.dy) + (int64_t)a.spos[i] * a.lddy;
#pragma unroll
      for (int c = 0; c < kMost; ++c)
        if (c < D) acc[c] += Elem<TI>::load(x + c);
    }
    float mine = 0.f;   // lane c: column c
#pragma unroll
    for (int c = 0; c < kMost; ++c) {
      const float s = any ? wave_sum(acc[c]) : 0.f;
      mine = lane == c ? s : mine;
    }
    if (lane < D) {
      TO* out = static_cast<TO*>(a.dw) + v * a.ldw + lane;
      *out = Elem<TO>::cast(a.accumulate ? __builtin_fmaf(mine, a.scale, Elem<TO>::load(out)) : mine * a.scale);
    }
  }
}

// Runs that cross tiles: the tile where a run begins adds its own partial row
// and those of the tiles that the run goes through, in order.  A wave looks at
// one tile and adds up to kFlight rows by itself; the waves of a workgroup
// share the longer runs that they found.
constexpr int kJoinWaves = 8;

// rows q0 .. q1 of a run that begins in `tile`
template <int N>
__device__ __forceinline__ void add_parts(const GradArgs& a, int64_t tile, int64_t q0, int64_t q1, int64_t from,
                                          float (&acc)[N]) {
  for (int64_t q = q0; q < q1; q += kFlight) {
    Cols<float, N> x[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const int64_t i = q + u < q1 ? q + u : q1 - 1;
      x[u].load(a.part + ((tile + i) * 2 + (i == 0 ? 1 : 0)) * a.D, from);
    }
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      if (q + u >= q1) break;
#pragma unroll
      for (int s = 0; s < N; ++s) acc[s] += x[u].get(s);
    }
  }
}

template <typename TI, typename TO>
__global__ __launch_bounds__(64 * kJoinWaves) void embed_grad_join(GradArgs a) {
  constexpr int N = Elem<TO>::kN;   // columns a lane
  __shared__ float sums[kJoinWaves - 1][64 * N];
  __shared__ int64_t rows[kJoinWaves];   // partial rows of the waves' longer runs, 0: none
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t slices = (a.D + 64 * N - 1) / (64 * N), tasks = a.tiles * slices;
  // a workgroup's waves take tasks far apart: a long run's slices go to as many workgroups
  const int64_t groups = (tasks + kJoinWaves - 1) / kJoinWaves;
  for (int64_t t0 = blockIdx.x; t0 < groups; t0 += gridDim.x) {
    int64_t m = 0;
    const int64_t t = t0 + w * groups, tile = t / slices, b = tile * a.tile, e = b + a.tile;
    if (t < tasks && e < a.n) {   // (nothing follows the last tile)
      const uint32_t key = a.skey[e - 1], next = a.skey[e], first = a.skey[b], front = b > 0 ? a.skey[b - 1] : ~0u;
      // a run crosses here, and it did not begin in an earlier tile
      if (key < (uint32_t)a.V && next == key && !(first == key && front == key)) {
        m = (first_not_before(a.skey, e, a.n, (int64_t)key + 1) - 1) / a.tile - tile + 1;
        if (m <= kFlight) {
          const int64_t c = ((t - tile * slices) * 64 + lane) * N, from = c + N <= a.D ? c : a.D - N;
          float acc[N] = {};
          add_parts<N>(a, tile, 0, m, from, acc);
          if (c < a.D) finish_row<TO, N>(a, key, c, from, acc);
          m = 0;
        }
      }
    }
    __syncthreads();   // the last round's rows and sums are read
    if (lane == 0) rows[w] = m;
    __syncthreads();
    for (int f = 0; f < kJoinWaves; ++f) {
      m = rows[f];
      if (m == 0) continue;   // (uniform)
      const int64_t t_f = t0 + f * groups, tile_f = t_f / slices;
      const int64_t c = ((t_f - tile_f * slices) * 64 + lane) * N, from = c + N <= a.D ? c : a.D - N;
      float acc[N] = {};
      add_parts<N>(a, tile_f, m * w / kJoinWaves, m * (w + 1) / kJoinWaves, from, acc);
      if (w > 0) {
#pragma unroll
        for (int s = 0; s < N; ++s) sums[w - 1][s * 64 + lane] = acc[s];
      }
      __syncthreads();
      if (w == 0 && c < a.D) {
#pragma unroll
        for (int q = 0; q < kJoinWaves - 1; ++q)
#pragma unroll
          for (int s = 0; s < N; ++s) acc[s] += sums[q][s * 64 + lane];
        finish_row<TO, N>(a, a.skey[(tile_f + 1) * a.tile], c, from, acc);
      }
      __syncthreads();
    }
  }
}

// Few tokens: a workgroup for each token and slice of columns looks for its
// token among all of them and, if it is the first such place, sums the rows in
// order: no sort, one launch, and one before it that zeroes the table.  1000
// tokens over 8192 x 1024 bf16: 10.3 us (sorted: 16.1), added to an fp32 table
// 6.3 (15.2); 777 of mixed frequency over 32003 x 1000 15.7 (22.3).  A token's
// rows are summed by one workgroup a slice however many they are, and where one
// token (a pad id of its own, a placeholder) is much of the batch that takes
// longer than the sort: a quarter, half, three quarters and all of the 777 21,
// 31, 40 and 48 us (23, 24, 24 and 24), of the 1000 12, 17, 24 and 29 (18, 19, 21
// and 20).
constexpr int kBriefTokens = 1024;
constexpr int64_t kBriefGroups = 4096;   // two rounds of the chip
constexpr int kBriefWaves = 8, kBriefFlight = 8;   // 4 waves: a run of 777 112 us; 16 rows in flight: 1000 x 1024 20

template <typename TI, typename TO>
__global__ __launch_bounds__(64 * kBriefWaves) void embed_grad_brief(GradArgs a, const void* __restrict__ tok,
                                                                     int wide) {
  constexpr int N = Elem<TI>::kN, kRounds = kBriefTokens / (64 * kBriefWaves);
  __shared__ int list[kBriefTokens];
  __shared__ int found[kBriefWaves];
  __shared__ float sums[kBriefWaves - 1][64 * N];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n = (int)a.n, slices = (int)a.slices;
  const int i = (int)blockIdx.x / slices;
  const int64_t c = ((int64_t)((int)blockIdx.x - i * slices) * 64 + lane) * N, from = c + N <= a.D ? c : a.D - N;
  const int64_t key = token_at(tok, wide, i);
  int64_t t[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int p = (w * kRounds + r) * 64 + lane;
    t[r] = token_at(tok, wide, p < n ? p : n - 1);
  }
  if (key < 0 || key >= a.V) return;
  unsigned long long same[kRounds];
  int count = 0;
  bool later = false;   // an earlier token is the same
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int p = (w * kRounds + r) * 64 + lane;
    same[r] = __ballot(p < n && t[r] == key);
    later = later || __ballot(p < i && t[r] == key) != 0;
    count += __popcll(same[r]);
  }
  if (lane == 0) found[w] = later ? -kBriefTokens : count;
  __syncthreads();
  int total = 0, at = 0;
#pragma unroll
  for (int q = 0; q < kBriefWaves; ++q) {
    at = q == w ? total : at;
    total += found[q];
  }
  if (total <= 0) return;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if ((same[r] >> lane) & 1) list[at + __popcll(same[r] & ((1ull << lane) - 1ull))] = (w * kRounds + r) * 64 + lane;
    at += __popcll(same[r]);
  }
  __syncthreads();
  const bool shared = total > kBriefFlight;   // (by the waves)
  const int first = shared ? total * w / kBriefWaves : 0;
  const int last = shared ? total * (w + 1) / kBriefWaves : w == 0 ? total : 0;
  float acc[N] = {};
  for (int q = first; q < last; q += kBriefFlight) {
    Cols<TI, N> x[kBriefFlight];
#pragma unroll
    for (int u = 0; u < kBriefFlight; ++u) {
      const int64_t row = __builtin_amdgcn_readfirstlane(list[q + u < last ? q + u : last - 1]);
      x[u].load(static_cast<const TI*>(a.dy) + row * a.lddy, from);
    }
#pragma unroll
    for (int u = 0; u < kBriefFlight; ++u) {
      if (q + u >= last) break;
#pragma unroll
      for (int s = 0; s < N; ++s) acc[s] += x[u].get(s);
    }
  }
  if (shared) {
    if (w > 0) {
#pragma unroll
      for (int s = 0; s < N; ++s) sums[w - 1][s * 64 + lane] = acc[s];
    }
    __syncthreads();
    if (w == 0) {
#pragma unroll
      for (int q = 0; q < kBriefWaves - 1; ++q)
#pragma unroll
        for (int s = 0; s < N; ++s) acc[s] += sums[q][s * 64 + lane];
    }
  }
  if (w == 0 && c < a.D) finish_row<TO, N>(a, key, c, from, acc);
}

// slices of a row of dY, 64 lanes' vectors each
int64_t lane_slices(int64_t D, int in_type) {
  const int64_t columns = 64 * (in_type == kF32 ? 4 : 8);
  return (D + columns - 1) / columns;
}

struct GradSizes {
  int64_t tile, tiles, sort_tiles, keys, cnt, slots, total;
  int bits, passes, rounds;
};

// Layout of the workspace: sorted keys and positions, slots, the same two again
// and digit counters for the radix passes, partial rows.
bool grad_sizes(int64_t n, int64_t V, int64_t D, int in_type, GradSizes& g) {
  if (n < 0 || n >= (1ll << 31) - (1 << 20) || V < 1 || V >= (1ll << 31) - 1 || D < 1) return false;
  int total_bits = 1;
  while ((V >> total_bits) != 0) ++total_bits;   // keys 0 .. V
  g.passes = (total_bits + kMaxBits - 1) / kMaxBits;
  g.bits = (total_bits + g.passes - 1) / g.passes;
  g.tile = tile_of(n * lane_slices(D, in_type));
  g.tiles = (n + g.tile - 1) / g.tile;
  g.rounds = n <= kFewTiles * 256 * kSmallRounds ? kSmallRounds : kLargeRounds;
  g.sort_tiles = (n + 256 * g.rounds - 1) / (256 * g.rounds);
  g.keys = (n + 63) / 64 * 64;
  g.cnt = n > kRankMax ? (g.sort_tiles << g.bits) : 0;
  const int64_t copies = n > kRankMax ? 2 : 1;
  g.slots = (V + 63) / 64 * 64;
  g.total = (g.keys * 2 * copies + g.slots + (g.cnt + 63) / 64 * 64 + g.tiles * 2 * D) * 4;
  return true;
}

bool is_brief(int64_t n, int64_t D, int in_type, int64_t ldw, int accumulate) {
  return n <= kBriefTokens && n * lane_slices(D, in_type) <= kBriefGroups && D >= kNarrow && (accumulate || ldw == D);
}

template <typename TI, typename TO>
int grad(GradArgs a, const void* tok, int wide, hipStream_t s) {
  if (a.brief) {
    const int64_t bytes = a.V * a.D * (int64_t)sizeof(TO);
    if (!a.accumulate)
      hipLaunchKernelGGL(embed_zero, dim3(groups_of((bytes + 4095) / 4096)), dim3(256), 0, s,
                         static_cast<uint16_t*>(a.dw), bytes);
    if (a.n > 0)
      hipLaunchKernelGGL((embed_grad_brief<TI, TO>), dim3((unsigned)(a.n * a.slices)),
                         dim3(64 * kBriefWaves), 0, s, a, tok, wide);
    SPMM_LAUNCH_CHECK();
    return 0;
  }
  if (a.D < kNarrow) {
    hipLaunchKernelGGL((embed_grad_narrow<TI, TO>), dim3(groups_of((a.V + 3) / 4)), dim3(256), 0, s, a);
    SPMM_LAUNCH_CHECK();
    return 0;
  }
  const int64_t row_bytes = a.D * (int64_t)sizeof(TO), groups = (a.tiles * a.slices + 3) / 4;
  const int64_t pieces = a.V * ((a.D / Elem<TO>::kN + 255) / 256);
  a.fill = row_bytes >= 2048 ? 0 : row_bytes * 64 <= kFillBytes ? 64 : kFillBytes / row_bytes;
  a.fills = a.fill ? (a.V + a.fill - 1) / a.fill : (pieces + 8 * kFillPieces - 1) / (8 * kFillPieces) * 8;
  if (a.accumulate || a.zeroed) a.fills = 0;
  if (groups + a.fills > 0)
    hipLaunchKernelGGL((embed_grad_sum<TI, TO>), dim3(groups_of(groups + a.fills)), dim3(256), 0, s, a);
  SPMM_LAUNCH_CHECK();
  if (a.tiles > 1) {
    const int64_t joins = a.tiles * ((a.D + 64 * Elem<TO>::kN - 1) / (64 * Elem<TO>::kN));
    hipLaunchKernelGGL((embed_grad_join<TI, TO>), dim3(groups_of((joins + kJoinWaves - 1) / kJoinWaves)),
                       dim3(64 * kJoinWaves), 0, s, a);
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

// bytes of workspace, or -1 for sizes that the kernels do not take; ldw: row stride of the table
SPMM_EXPORT int64_t spmm_embedding_grad_ws(int64_t n, int64_t V, int64_t D, int in_type, int64_t ldw, int accumulate) {
  GradSizes g;
  if (!grad_sizes(n, V, D, in_type, g)) return -1;
  return is_brief(n, D, in_type, ldw, accumulate) ? 0 : g.total;
}

SPMM_EXPORT int spmm_embedding_grad(const void* dy, int64_t lddy, int in_type, const void* tok, int wide, int64_t n,
                                    int64_t V, int64_t D, float scale, void* dw, int64_t ldw, int out_type,
                                    int accumulate, void* ws, int64_t ws_bytes, hipStream_t s) {
  GradSizes g;
  if (!grad_sizes(n, V, D, in_type, g)) return (int)hipErrorInvalidValue;
  const bool brief = is_brief(n, D, in_type, ldw, accumulate);
  if (!brief && ws_bytes < g.total) return (int)hipErrorInvalidValue;
  uint32_t* ka = static_cast<uint32_t*>(ws);   // (all null in a brief call, which uses none of it)
  int32_t* pa = reinterpret_cast<int32_t*>(ka + g.keys);
  uint32_t* skey = ka;
  int32_t* spos = pa;
  int32_t* slot = accumulate ? nullptr : pa + g.keys;
  char* behind = reinterpret_cast<char*>(pa + g.keys + g.slots);
  int64_t zeroed = 0;   // bytes of the table that the sort's launch zeroes
  if (brief) {
    // no sort
  } else if (n > kRankMax) {
    uint32_t* kb = reinterpret_cast<uint32_t*>(behind);
    int32_t* pb = reinterpret_cast<int32_t*>(kb + g.keys);
    int32_t* cnt = pb + g.keys;
    behind = reinterpret_cast<char*>(cnt + (g.cnt + 63) / 64 * 64);
    const uint32_t* kin = nullptr;
    const int32_t* pin = nullptr;
    uint32_t* kout = ka;
    int32_t* pout = pa;
    const bool scan = g.sort_tiles > kFewTiles;
    const dim3 grid((unsigned)g.sort_tiles);
    for (int p = 0; p < g.passes; ++p) {
      const int shift = p * g.bits;
      hipLaunchKernelGGL(embed_digit_count, grid, dim3(256), 0, s, tok, wide, kin, n, V, shift, g.bits, g.rounds, cnt);
      if (scan) hipLaunchKernelGGL(embed_digit_scan, dim3(1), dim3(1024), 0, s, cnt, g.sort_tiles, g.bits);
      auto scatter = g.rounds == kSmallRounds ? embed_digit_scatter<kSmallRounds> : embed_digit_scatter<kLargeRounds>;
      hipLaunchKernelGGL(scatter, grid, dim3(256), 0, s, tok, wide, kin, pin, n, V, shift, g.bits, g.sort_tiles,
                         (int)scan, cnt, kout, pout, p == g.passes - 1 ? slot : nullptr);
      kin = kout;
      pin = pout;
      kout = kout == ka ? kb : ka;
      pout = pout == pa ? pb : pa;
    }
    skey = const_cast<uint32_t*>(kin);
    spos = const_cast<int32_t*>(pin);
  } else if (n > 0) {
    const int64_t row_bytes = D * (out_type == kF32 ? 4 : 2);
    if (!accumulate && D >= kNarrow && ldw == D && n * kFewRows <= V) zeroed = V * row_bytes;
    const int64_t fills = (zeroed + 16 * 64 * kRankWaves - 1) / (16 * 64 * kRankWaves);
    hipLaunchKernelGGL(embed_rank_sort, dim3((unsigned)((n + 63) / 64) + (zeroed ? groups_of(fills) : 0)),
                       dim3(64 * kRankWaves), 0, s, tok, wide, (int)n, V, skey, spos, zeroed ? nullptr : slot,
                       static_cast<uint16_t*>(dw), zeroed);
  }
  SPMM_LAUNCH_CHECK();
  GradArgs a;
  a.dy = dy;
  a.lddy = lddy;
  a.skey = skey;
  a.spos = spos;
  a.slot = slot;
  a.n = n;
  a.V = V;
  a.D = D;
  a.ldw = ldw;
  a.tile = g.tile;
  a.tiles = g.tiles;
  a.scale = scale;
  a.dw = dw;
  a.part = reinterpret_cast<float*>(behind);
  a.accumulate = accumulate;
  a.zeroed = zeroed != 0;
  a.slices = lane_slices(D, in_type);
  a.brief = brief;
  SPMM_VOCAB_TYPE(in_type, TI, {
    if (out_type == kF32) return grad<TI, float>(a, tok, wide, s);
    if (out_type == in_type) return grad<TI, TI>(a, tok, wide, s);
    return (int)hipErrorInvalidValue;
  });
  return 0;
}
