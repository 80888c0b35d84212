// A token from a row of logits: temperature, top-k, top-p, min-p and a given uniform number.
//
// With l the logits, M their largest and w_i = exp((l_i - M) / T), the entries are walked from the largest logit down (equal
// ones by their index): the first top_k of them, of those the shortest prefix that holds top_p of their mass, of those the
// ones with w >= min_p.  What is kept is a prefix, of mass S; the answer is its first entry whose mass, with all before it,
// exceeds u * S.  So four questions have to be answered, and nothing is sorted: the mass of the k largest, the mass at which
// top_p is reached, the mass of the entries with w >= min_p, and the entry at a given mass.
//
// Masses are whole numbers: w * 2^44 to the nearest (u64, at most 2^19 entries).  Their sums do not depend on the order in
// which threads add them, so a row's answer is the same on every run, and a draw falls on the side of a border that 64-bit
// sums give (a rounding is 2^-45 of the largest weight; f32 weights would move one draw in 10^4 at 10^5 undecided entries).
#include "st_common.h"

namespace {

constexpr int NBIN = 2048;
constexpr double ONE = 17592186044416.0;   // 2^44

// ascending order of keys = descending order of logits; -0 and 0 are one value
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l + 0.0f);
  return (b >> 31) ? b : ~(b | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float((k >> 31) ? k : ~k & 0x7fffffffu); }

struct Row {
  double top, inv_t;
};
__device__ __forceinline__ double weight(const Row& r, float l) {
  if ((double)l == r.top) return 1.0;
  const double z = ((double)l - r.top) * r.inv_t;
  return z <= 0.0 ? exp(z) : 0.0;   // not for a NaN: a finite logit under an infinite one at an infinite temperature
}
__device__ __forceinline__ unsigned long long mass(double w) { return (unsigned long long)(w * ONE + 0.5); }

template <int TYPE> struct LOf;
template <> struct LOf<ST_TYPE_F32> { typedef float t; };
template <> struct LOf<ST_TYPE_BF16> { typedef uint16_t t; };
template <> struct LOf<ST_TYPE_F16> { typedef _Float16 t; };
template <int TYPE> __device__ __forceinline__ float logit(typename LOf<TYPE>::t v) {   // NaN: no entry
  float f;
  if constexpr (TYPE == ST_TYPE_BF16) f = __uint_as_float((uint32_t)v << 16);
  else f = (float)v;
  return f == f ? f : -INFINITY;
}

__device__ __forceinline__ float setting(const float* rows, float all, int s) { return rows ? rows[s] : all; }

template <class T> __device__ __forceinline__ T block_sum(T v, T* part, int n_waves) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  T s = 0;
  for (int i = 0; i < n_waves; ++i) s += part[i];
  return s;
}

// The entry at which the count (or the mass) of the walk first exceeds `target`: its key, and what lies before the entries that
// share the key.  Three rounds over the row: 11, 11 and 10 bits of the key.
struct Found {
  uint32_t key;
  uint32_t count;
  unsigned long long mass;
};
struct Hist {
  unsigned long long mass[NBIN];
  uint32_t count[NBIN];
  unsigned long long wave_mass[16];
  uint32_t wave_count[16];
  Found found;
};

template <int TYPE, bool BY_COUNT>
__device__ Found descend(const typename LOf<TYPE>::t* row, int V, const Row& r, unsigned long long target, Hist& h) {
  Found f = {0, 0, 0};
  const int nt = blockDim.x, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int per = NBIN / nt;
  for (int round = 0; round < 3; ++round) {
    const int low = round == 0 ? 21 : round == 1 ? 10 : 0, bits = round == 2 ? 10 : 11;
    for (int i = threadIdx.x; i < NBIN; i += nt) h.mass[i] = 0, h.count[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += nt) {
      const float l = logit<TYPE>(row[i]);
      if (l == -INFINITY) continue;
      const uint32_t k = key_of(l);
      if (round > 0 && (k >> (low + bits)) != (f.key >> (low + bits))) continue;
      const int bin = (k >> low) & ((1 << bits) - 1);
      atomicAdd(&h.count[bin], 1u);
      atomicAdd(&h.mass[bin], mass(weight(r, l)));
    }
    __syncthreads();
    uint32_t c = 0;
    unsigned long long m = 0;
    for (int i = 0; i < per; ++i) c += h.count[threadIdx.x * per + i], m += h.mass[threadIdx.x * per + i];
    uint32_t ci = c;
    unsigned long long mi = m;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t cu = __shfl_up(ci, o, 64);
      const unsigned long long mu = __shfl_up(mi, o, 64);
      if (lane >= o) ci += cu, mi += mu;
    }
    if (lane == 63) h.wave_count[wv] = ci, h.wave_mass[wv] = mi;
    __syncthreads();
    c = ci - c + f.count;
    m = mi - m + f.mass;
    for (int i = 0; i < wv; ++i) c += h.wave_count[i], m += h.wave_mass[i];
    for (int i = 0; i < per; ++i) {
      const int bin = threadIdx.x * per + i;
      const bool here = BY_COUNT ? c <= target && target < (unsigned long long)c + h.count[bin] : m <= target && target < m + h.mass[bin];
      if (here) h.found = Found{f.key | ((uint32_t)bin << low), c, m};
      c += h.count[bin];
      m += h.mass[bin];
    }
    __syncthreads();
    f = h.found;
    __syncthreads();
  }
  return f;
}

// One workgroup a row.
template <int TYPE> __global__ __launch_bounds__(1024) void sample_row_kernel(SampleArgs a) {
  typedef typename LOf<TYPE>::t T;
  __shared__ Hist h;
  __shared__ float red[16];
  __shared__ int at[16];
  const int b = blockIdx.x;
  if (a.n_dev && b >= *a.n_dev) return;
  const int s = a.idx ? a.idx[b] : b;
  const T* row = (const T*)a.logits + (size_t)b * a.ld;
  const int nt = blockDim.x, nw = nt >> 6, lane = threadIdx.x & 63, wv = threadIdx.x >> 6, V = a.V;
  float top = -INFINITY;
  for (int i = threadIdx.x; i < V; i += nt) top = fmaxf(top, logit<TYPE>(row[i]));
  top = wave_max(top);
  if (lane == 0) red[wv] = top;
  __syncthreads();
  for (int i = 0; i < nw; ++i) top = fmaxf(top, red[i]);
  if (top == -INFINITY) {
    if (threadIdx.x == 0) {
      a.ids[b] = -1;
      if (a.logp) a.logp[b] = -INFINITY;
    }
    return;
  }
  const float temp = setting(a.set.temperature_rows, a.set.temperature, s);
  const int top_k = a.set.top_k_rows ? a.set.top_k_rows[s] : a.set.top_k;
  const float top_p = setting(a.set.top_p_rows, a.set.top_p, s), min_p = setting(a.set.min_p_rows, a.set.min_p, s);
  const bool greedy = !(temp > 0.0f) || top_k == 1;
  Found f = {key_of(top), 0, 0};
  uint32_t nth = 0;
  double w = 1.0, total = 1.0;
  if (!greedy) {
    Row r = {(double)top, 1.0 / (double)temp};
    unsigned long long all = 0, over = 0;
    uint32_t n = 0;
    for (int i = threadIdx.x; i < V; i += nt) {
      const float l = logit<TYPE>(row[i]);
      if (l == -INFINITY) continue;
      const double x = weight(r, l);
      ++n;
      all += mass(x);
      if (x >= (double)min_p) over += mass(x);
    }
    n = block_sum<uint32_t>(n, h.wave_count, nw);
    all = block_sum<unsigned long long>(all, h.wave_mass, nw);
    over = block_sum<unsigned long long>(over, h.wave_mass, nw);
    unsigned long long S = all;
    if (top_k > 0 && (uint32_t)top_k < n) {
      f = descend<TYPE, true>(row, V, r, (unsigned long long)(top_k - 1), h);
      S = f.mass + (top_k - f.count) * mass(weight(r, of_key(f.key)));
    }
    if (top_p < 1.0f) {
      const double want = ceil((double)top_p * (double)S);
      const unsigned long long t = want < 1.0 ? 0ull : (unsigned long long)want - 1ull;
      f = descend<TYPE, false>(row, V, r, t, h);
      const unsigned long long one = mass(weight(r, of_key(f.key)));
      S = f.mass + ((t - f.mass) / one + 1) * one;
    }
    if (min_p > 0.0f && over < S) S = over;
    const unsigned long long first = mass(1.0);
    if (S < first) S = first;   // the largest entry stays whatever is asked
    const double u = fmin(fmax((double)a.u[(size_t)s * a.u_stride], 0.0), 1.0);
    unsigned long long t = (unsigned long long)(u * (double)S);
    if (t >= S) t = S - 1;
    f = descend<TYPE, false>(row, V, r, t, h);
    w = weight(r, of_key(f.key));
    nth = (uint32_t)((t - f.mass) / mass(w));
    total = (double)S / ONE;
  }
  // the entry is the nth by index among those of its key: counts of every thread's stretch of the row
  const int stretch = (V + nt - 1) / nt, i0 = min(V, (int)threadIdx.x * stretch), i1 = min(V, i0 + stretch);
  int n = 0;
  for (int i = i0; i < i1; ++i) {
    const float l = logit<TYPE>(row[i]);
    n += l > -INFINITY && key_of(l) == f.key;
  }
  int incl = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(incl, o, 64);
    if (lane >= o) incl += v;
  }
  if (lane == 63) at[wv] = incl;
  __syncthreads();
  int before = incl - n;
  for (int i = 0; i < wv; ++i) before += at[i];
  if ((int)nth >= before && (int)nth < before + n) {
    for (int i = i0; i < i1; ++i) {
      const float l = logit<TYPE>(row[i]);
      if (l > -INFINITY && key_of(l) == f.key && before++ == (int)nth) {
        a.ids[b] = i;
        if (a.logp) a.logp[b] = (float)log(w / total);
      }
    }
  }
}

}  // namespace

size_t sample_workspace(int, int) { return 0; }

int sample_check(const StSampleSettings* s) {
  ST_CHECK_ARG(s != nullptr, "settings struct is NULL");
  ST_CHECK_ARG(s->temperature_rows || (s->temperature >= 0.0f && s->temperature < INFINITY), "temperature=%g must be finite and not negative", s->temperature);
  ST_CHECK_ARG(s->top_k_rows || s->top_k >= 0, "top_k=%d must not be negative (0: off)", s->top_k);
  ST_CHECK_ARG(s->top_p_rows || (s->top_p > 0.0f && s->top_p <= 1.0f), "top_p=%g must lie in (0, 1]", s->top_p);
  ST_CHECK_ARG(s->min_p_rows || (s->min_p >= 0.0f && s->min_p <= 1.0f), "min_p=%g must lie in [0, 1]", s->min_p);
  return ST_OK;
}

int sample_launch(const SampleArgs& a, hipStream_t st) {
  const dim3 grid(a.B), block(1024);
  if (a.type == ST_TYPE_F32) hipLaunchKernelGGL(sample_row_kernel<ST_TYPE_F32>, grid, block, 0, st, a);
  else if (a.type == ST_TYPE_BF16) hipLaunchKernelGGL(sample_row_kernel<ST_TYPE_BF16>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(sample_row_kernel<ST_TYPE_F16>, grid, block, 0, st, a);
  ST_LAUNCH_CHECK();
  return ST_OK;
}

extern "C" size_t st_sample_workspace_bytes(int B, int V) { return B > 0 && V > 0 && V <= ST_SAMPLE_MAX_VOCAB ? sample_workspace(B, V) : 0; }

extern "C" int st_sample_logits(const void* logits, int type, int64_t ld, int B, int V, const float* u, const StSampleSettings* settings,
                                int32_t* ids, float* logp, void* workspace, size_t workspace_bytes, void* stream) {
  ST_TRY(sample_check(settings));
  ST_CHECK_ARG(type == ST_TYPE_F32 || type == ST_TYPE_BF16 || type == ST_TYPE_F16, "type=%d unknown", type);
  ST_CHECK_ARG(B >= 0, "B=%d", B);
  ST_CHECK_ARG(V >= 1 && V <= ST_SAMPLE_MAX_VOCAB, "V=%d (1 .. %d)", V, ST_SAMPLE_MAX_VOCAB);
  if (B == 0) return ST_OK;
  ST_CHECK_ARG(logits && u && ids, "NULL buffer");
  ST_CHECK_ARG(((size_t)logits & (type == ST_TYPE_F32 ? 3 : 1)) == 0, "logits must lie on their type's size");
  ST_CHECK_ARG(ld >= 0, "ld=%lld", (long long)ld);
  const size_t need = sample_workspace(B, V);
  if (need > workspace_bytes || (need && !workspace)) {
    st_set_error("workspace too small: need %zu bytes, have %zu", need, workspace ? workspace_bytes : (size_t)0);
    return ST_ENOMEM;
  }
  SampleArgs a = {};
  a.logits = logits; a.type = type; a.ld = ld; a.B = B; a.V = V; a.u = u; a.u_stride = 1; a.set = *settings;
  a.ids = ids; a.logp = logp; a.ws = workspace;
  return sample_launch(a, (hipStream_t)stream);
}
