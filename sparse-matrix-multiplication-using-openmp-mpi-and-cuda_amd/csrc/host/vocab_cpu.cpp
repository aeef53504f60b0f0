// CPU engine of the operators on rows over a vocabulary (embedding lookup and
// gradient, token log-probabilities, distillation): the definitions that the
// gfx950 kernels of embedding.hip and vocab_logits.hip follow, in double inside
// and fp32 at the borders, OpenMP over rows.
#include <omp.h>

#include <algorithm>
#include <cerrno>
#include <cmath>
#include <cstdint>
#include <limits>
#include <new>
#include <numeric>
#include <vector>

#define SPMM_HOST_EXPORT extern "C" __attribute__((visibility("default")))

namespace {

constexpr double kNoMass = -std::numeric_limits<double>::infinity();
const float kNan = std::numeric_limits<float>::quiet_NaN();

inline int threads_or_default(int n) { return n > 0 ? n : omp_get_max_threads(); }

// One scratch row of n elements for every thread, allocated before the threads
// start: false (and no exception, which a C caller could not take) if there is
// no memory for them.
template <typename T>
struct Scratch {
  std::vector<T> rows;
  size_t n = 0;
  bool make(int threads, int64_t width) noexcept {
    n = (size_t)width;
    try {
      rows.resize((size_t)threads * n);
    } catch (const std::exception&) {
      return false;
    }
    return true;
  }
  T* mine() { return rows.data() + (size_t)omp_get_thread_num() * n; }
};

// maximum of the numbers (a NaN is passed over; it reaches the sum), and the sum of exp((z - m) / T)
struct RowSum {
  double m, z, u;
};
inline double origin(double m) { return m == kNoMass ? 0.0 : m; }
inline RowSum row_sum(const float* z, int64_t V, double inv_t) {
  double m = kNoMass;
  for (int64_t j = 0; j < V; ++j)
    if (z[j] > m) m = z[j];
  const double o = origin(m);
  double s = 0, u = 0;
  for (int64_t j = 0; j < V; ++j) {
    const double t = (z[j] - o) * inv_t, e = std::exp(t);
    s += e;
    if (e != 0) u += e * t;
  }
  return RowSum{m, s, u};
}

// larger logits first (NaN above all), then lower columns
inline bool before(const float* z, int32_t a, int32_t b) {
  const bool na = std::isnan(z[a]), nb = std::isnan(z[b]);
  if (na != nb) return na;
  if (!na && z[a] != z[b]) return z[a] > z[b];
  return a < b;
}

}  // namespace

SPMM_HOST_EXPORT int spmm_cpu_embedding(int64_t n, int64_t V, int64_t D, const float* W, const int64_t* tok,
                                        double scale, float* Y, int nthreads) {
#pragma omp parallel for num_threads(threads_or_default(nthreads))
  for (int64_t i = 0; i < n; ++i) {
    const int64_t t = tok[i];
    float* y = Y + i * D;
    if (t >= 0 && t < V) {
      for (int64_t d = 0; d < D; ++d) y[d] = (float)(W[t * D + d] * scale);
    } else {
      std::fill(y, y + D, t == -1 ? 0.f : kNan);
    }
  }
  return 0;
}

// dW (fp32, given) += scale * S^T dY
SPMM_HOST_EXPORT int spmm_cpu_embedding_grad(int64_t n, int64_t V, int64_t D, const float* dY, const int64_t* tok,
                                             double scale, float* dW, int nthreads) {
  const int threads = threads_or_default(nthreads);
  std::vector<int64_t> pos, start;   // positions by token; the first of each run of equal tokens
  Scratch<double> scratch;
  try {
    for (int64_t i = 0; i < n; ++i)
      if (tok[i] >= 0 && tok[i] < V) pos.push_back(i);
    std::stable_sort(pos.begin(), pos.end(), [&](int64_t a, int64_t b) { return tok[a] < tok[b]; });
    for (size_t i = 0; i < pos.size(); ++i)
      if (i == 0 || tok[pos[i]] != tok[pos[i - 1]]) start.push_back((int64_t)i);
    start.push_back((int64_t)pos.size());
  } catch (const std::exception&) {
    return ENOMEM;
  }
  if (!scratch.make(threads, D)) return ENOMEM;
#pragma omp parallel for schedule(dynamic, 16) num_threads(threads)
  for (int64_t r = 0; r < (int64_t)start.size() - 1; ++r) {
    double* acc = scratch.mine();
    std::fill(acc, acc + D, 0.0);
    for (int64_t i = start[(size_t)r]; i < start[(size_t)r + 1]; ++i) {
      const float* x = dY + pos[(size_t)i] * D;
      for (int64_t d = 0; d < D; ++d) acc[d] += x[d];
    }
    float* w = dW + tok[pos[(size_t)start[(size_t)r]]] * D;
    for (int64_t d = 0; d < D; ++d) w[d] = (float)(w[d] + acc[d] * scale);
  }
  return 0;
}

// stat: [4][n] log-probability, entropy, maximum, Z.  top_col / top_val: [n][k].
SPMM_HOST_EXPORT int spmm_cpu_token_logprobs(int64_t n, int64_t V, const float* z, const int64_t* tok, double inv_t,
                                             int k, float* stat, int32_t* top_col, float* top_val, int nthreads) {
  const int threads = threads_or_default(nthreads);
  Scratch<int32_t> scratch;
  if (!scratch.make(threads, k > 0 ? V : 0)) return ENOMEM;
#pragma omp parallel for num_threads(threads)
  for (int64_t i = 0; i < n; ++i) {
    const float* zi = z + i * V;
    const RowSum r = row_sum(zi, V, inv_t);
    const double o = origin(r.m), logz = r.z == 0 ? 0.0 : std::log(r.z);
    const int64_t t = tok[i];
    stat[i] = t >= 0 && t < V ? (float)((zi[t] - o) * inv_t - logz) : (t == -1 ? 0.f : kNan);
    stat[n + i] = r.z == 0 ? 0.f : (float)(logz - r.u / r.z);
    stat[2 * n + i] = (float)r.m;
    stat[3 * n + i] = (float)r.z;
    if (k > 0) {
      int32_t* idx = scratch.mine();
      std::iota(idx, idx + V, 0);
      std::partial_sort(idx, idx + k, idx + V, [&](int32_t a, int32_t b) { return before(zi, a, b); });
      for (int j = 0; j < k; ++j) {
        top_col[i * k + j] = idx[j];
        top_val[i * k + j] = (float)((zi[idx[j]] - o) * inv_t - logz);
      }
    }
  }
  return 0;
}

SPMM_HOST_EXPORT int spmm_cpu_token_logprobs_grad(int64_t n, int64_t V, const float* z, const int64_t* tok, double inv_t,
                                                  const float* stat, const float* g, const float* h, float* out,
                                                  int nthreads) {
#pragma omp parallel for num_threads(threads_or_default(nthreads))
  for (int64_t i = 0; i < n; ++i) {
    const float* zi = z + i * V;
    float* oi = out + i * V;
    const int64_t t = tok[i];
    double gi = g && t != -1 ? g[i] * inv_t : 0.0;
    const double hi = h ? h[i] * inv_t : 0.0;
    if (gi == 0 && hi == 0) {
      std::fill(oi, oi + V, 0.f);
      continue;
    }
    if (t < -1 || t >= V) gi = kNan;
    const RowSum r = row_sum(zi, V, inv_t);
    const double o = origin(r.m), logz = r.z == 0 ? 0.0 : std::log(r.z);
    for (int64_t j = 0; j < V; ++j) {
      const double lq = (zi[j] - o) * inv_t - logz, q = std::exp(lq);
      oi[j] = (float)((j == t ? gi : 0.0) - gi * q - (q == 0 ? 0.0 : hi * q * (lq + stat[n + i])));
    }
  }
  return 0;
}

// Teacher entries with column -1 are absent; one outside the vocabulary, or of a
// value of NaN or +inf, makes the row's loss and gradient NaN.  out (null: loss only) may be z itself.
SPMM_HOST_EXPORT int spmm_cpu_distill(int64_t n, int64_t V, const float* z, const int64_t* rowptr, const int32_t* col,
                                      const float* val, int64_t nnz, double inv_t, float* loss, float* stat,
                                      const float* weight, float* out, int nthreads) {
  const int threads = threads_or_default(nthreads);
  Scratch<double> scratch;
  if (!scratch.make(threads, out ? V : 0)) return ENOMEM;
#pragma omp parallel for num_threads(threads)
  for (int64_t i = 0; i < n; ++i) {
    double* p = scratch.mine();
    const float* zi = z + i * V;
    const int64_t b = std::min(std::max<int64_t>(rowptr[i], 0), nnz);
    const int64_t e = std::min(std::max(rowptr[i + 1], b), nnz);
    double tm = kNoMass, ts = 0;
    bool bad = false;
    for (int64_t k = b; k < e; ++k) {
      bad |= col[k] < -1 || col[k] >= V;
      if (col[k] != -1 && val[k] > tm) tm = val[k];
    }
    const double to = origin(tm);
    for (int64_t k = b; k < e; ++k)
      if (col[k] != -1) ts += std::exp((val[k] - to) * inv_t);
    bad |= ts != ts;
    const RowSum r = row_sum(zi, V, inv_t);
    const double o = origin(r.m), logz = r.z == 0 ? 0.0 : std::log(r.z);
    double l = 0;
    if (out) std::fill(p, p + V, 0.0);
    if (ts != 0 && !bad)
      for (int64_t k = b; k < e; ++k) {
        if (col[k] == -1) continue;
        const double u = (val[k] - to) * inv_t, pk = std::exp(u) / ts;
        if (pk != 0) l += pk * ((u - std::log(ts)) - ((zi[col[k]] - o) * inv_t - logz));
        if (out) p[col[k]] += pk;
      }
    loss[i] = bad ? kNan : (float)l;
    stat[4 * i] = (float)r.m;
    stat[4 * i + 1] = bad ? kNan : (float)r.z;
    stat[4 * i + 2] = (float)to;
    stat[4 * i + 3] = bad ? kNan : (float)ts;
    if (!out) continue;
    const double w = (weight ? weight[i] : 1.0) * inv_t;
    float* oi = out + i * V;
    if (w == 0 || (ts == 0 && !bad)) {
      std::fill(oi, oi + V, 0.f);
      continue;
    }
    for (int64_t j = 0; j < V; ++j)
      oi[j] = bad ? kNan : (float)(w * ((r.z == 0 ? 0.0 : std::exp((zi[j] - o) * inv_t) / r.z) - p[j]));
  }
  return 0;
}
