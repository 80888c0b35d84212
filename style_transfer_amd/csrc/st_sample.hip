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

// Everything below is inlined into its kernel and shared memory is reached by its own instructions: passing it to functions by
// reference makes flat accesses of it, and code of many times the size.
#define SM_INLINE __attribute__((always_inline))

typedef unsigned long long u64;

constexpr double ONE = 17592186044416.0;   // 2^44
constexpr u64 ONE_MASS = 1ull << 44;

// ---- values ----------------------------------------------------------------------------------------------------------------
template <int TYPE> struct LOf;
template <> struct LOf<ST_TYPE_F32> { typedef float t; };
template <> struct LOf<ST_TYPE_BF16> { typedef uint16_t t; };
template <> struct LOf<ST_TYPE_F16> { typedef _Float16 t; };
template <int TYPE> __device__ __forceinline__ float logit(typename LOf<TYPE>::t v) {   // -inf: no entry (a NaN is none either)
  float f;
  if constexpr (TYPE == ST_TYPE_BF16) f = __uint_as_float((uint32_t)v << 16);
  else f = (float)v;
  return f == f ? f : -INFINITY;
}

// ascending keys are descending logits; -0 and 0 are one value.  An entry's place in the walk is (key, index) in one number.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l + 0.0f);
  return (b >> 31) ? b : ~(b | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float((k >> 31) ? k : ~k & 0x7fffffffu); }
__device__ __forceinline__ u64 place_of(float l, int i) { return (u64)key_of(l) << 32 | (uint32_t)i; }

struct Scale {
  float top;
  double inv_t;   // log2(e) / temperature
};
// exp((l - top) / T) to about 2^-43 of the value: 2^y with y = n + f, |f| <= 1/2, the series of 2^f to the 11th power (the 12th
// term is below 1e-14).  Half the instructions of the library's exp, which is good to the last bit.
__device__ __forceinline__ double weight(const Scale& c, float l) {
#pragma clang fp contract(off)   // the same value wherever it is computed: bins and the entries found in them have to agree
  double y = l == c.top ? 0.0 : ((double)l - (double)c.top) * c.inv_t;
  y = fmax(y, -1000.0);
  const double n = rint(y), f = y - n;
  double p = 4.44553827187081e-10;              // ln(2)^k / k!, k = 11 .. 0
  p = fma(p, f, 7.054911620801121e-09);
  p = fma(p, f, 1.0178086009239696e-07);
  p = fma(p, f, 1.3215486790144305e-06);
  p = fma(p, f, 1.5252733804059838e-05);
  p = fma(p, f, 1.5403530393381606e-04);
  p = fma(p, f, 1.3333558146428441e-03);
  p = fma(p, f, 9.618129107628477e-03);
  p = fma(p, f, 5.5504108664821576e-02);
  p = fma(p, f, 2.402265069591007e-01);
  p = fma(p, f, 6.931471805599453e-01);
  p = fma(p, f, 1.0);
  return ldexp(p, (int)n);
}
// w in units of 2^-44: added to 2^52 it stands in the low bits of the sum
__device__ __forceinline__ u64 mass_of(double w) {
  return (u64)__double_as_longlong(fma(w, ONE, 4503599627370496.0)) & 0xfffffffffffffull;
}

// ---- the row ---------------------------------------------------------------------------------------------------------------
// 16-byte chunks on the row's own alignment: chunk c holds the entries c * EPC - pad + 0..EPC-1.
template <int TYPE> struct Row {
  typedef typename LOf<TYPE>::t T;
  static constexpr int EPC = 16 / sizeof(T);
  const T* p;          // entry 0
  int n, pad, chunks;
  __device__ __forceinline__ Row(const T* p_, int n_) : p(p_), n(n_) {
    pad = (int)(((size_t)p & 15) / sizeof(T));
    chunks = (n + pad + EPC - 1) / EPC;
  }
  // entry j of a chunk, as f32 (a NaN stays one)
  static __device__ __forceinline__ float entry(f32x4 k, int j) {
    if constexpr (TYPE == ST_TYPE_F32) return k[j];
    else if constexpr (TYPE == ST_TYPE_F16) return (float)__builtin_bit_cast(h8, k)[j];
    else return __uint_as_float(j & 1 ? __float_as_uint(k[j >> 1]) & 0xffff0000u : __float_as_uint(k[j >> 1]) << 16);
  }
  // the same where j is not known to hipcc
  static __device__ __forceinline__ float pick(f32x4 k, int j) {
    const int w = TYPE == ST_TYPE_F32 ? j : j >> 1;
    const float v = w & 2 ? (w & 1 ? k[3] : k[2]) : (w & 1 ? k[1] : k[0]);
    if constexpr (TYPE == ST_TYPE_F32) return v;
    const uint32_t u = j & 1 ? __float_as_uint(v) >> 16 : __float_as_uint(v) & 0xffffu;
    if constexpr (TYPE == ST_TYPE_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)u);
    else return __uint_as_float(u << 16);
  }
  // a chunk that sticks out of the row, put together from single entries; -inf outside
  __device__ __forceinline__ f32x4 edge(int c) const {
    f32x4 k;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if constexpr (TYPE == ST_TYPE_F32) {
        const int i = c * 4 - pad + w;
        k[w] = i >= 0 && i < n ? p[i] : -INFINITY;
      } else {
        uint32_t u = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = c * 8 - pad + 2 * w + h;
          const uint32_t v = i >= 0 && i < n ? (uint32_t)((const uint16_t*)p)[i] : TYPE == ST_TYPE_F16 ? 0xfc00u : 0xff80u;
          u |= v << (16 * h);
        }
        k[w] = __uint_as_float(u);
      }
    }
    return k;
  }
  // f(chunk, number) for this thread's chunks, LOADS of them under way at a time.  A row is read again for each pass: it comes from
  // the L2 or the last-level cache then, and with the workgroups that shared memory leaves room for that is faster than one copy of
  // the row in shared memory (1024 x 19724: 69 us against 93) or in registers (98).
  template <int LOADS, class F> __device__ __forceinline__ void each(F f) const {
    const int first = pad ? 1 : 0, last = (n + pad) / EPC, nt = blockDim.x;   // [first, last): in the row as a whole
    const f32x4* q = (const f32x4*)(p - pad);
#pragma unroll 1
    for (int c = first + (int)threadIdx.x; c < last; c += LOADS * nt) {
      f32x4 k[LOADS];
#pragma unroll
      for (int u = 0; u < LOADS; ++u) k[u] = q[min(c + u * nt, last - 1)];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < LOADS; ++u)
        if (c + u * nt < last) f(k[u], c + u * nt);
    }
    const int t = nt - 1 - (int)threadIdx.x;   // the last threads have the least to do
    const int c = t == 0 && first ? 0 : t == 1 && last >= first && last < chunks ? last : -1;
    if (c >= 0) f(edge(c), c);
  }
  // f(logit, index) for the entries above -inf of which yes(logit) holds (it may hold for a NaN or -inf)
  template <int LOADS, class Y, class F> __device__ __forceinline__ void each_if(Y yes, F f) const {
    each<LOADS>([&](f32x4 k, int c) SM_INLINE {
      uint32_t hits = 0;
#pragma unroll
      for (int j = 0; j < EPC; ++j) hits |= (uint32_t)yes(entry(k, j)) << j;
      while (hits) {
        const int j = __builtin_ctz(hits);
        hits &= hits - 1;
        const float l = pick(k, j);
        if (l > -INFINITY) f(l, c * EPC + j - pad);
      }
    });
  }
};

// ---- sums over the workgroup ---------------------------------------------------------------------------------------------
struct Shared {
  u64 digit_mass[256];
  uint32_t digit_count[256];
  u64 wave_u64[16], wave_any[16], wave_all[16];
  uint32_t wave_u32[16];
  float wave_f[32];
  u64 found_place, found_mass;
  uint32_t found_count, found_bin, n;
  uint32_t part_end[32], part_at[32];
};

// Sums over the lanes up to this one, by row shifts and row broadcasts: no way through shared memory
#define SM_DPP(v, ctrl, rows) __builtin_amdgcn_update_dpp(0, (int)(v), ctrl, rows, 0xf, false)
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v += SM_DPP(v, 0x111, 0xf);   // row_shr:1, 2, 4, 8 (lanes from outside a row of 16 count 0)
  v += SM_DPP(v, 0x112, 0xf);
  v += SM_DPP(v, 0x114, 0xf);
  v += SM_DPP(v, 0x118, 0xf);
  v += SM_DPP(v, 0x142, 0xa);   // row_bcast:15 into rows 1 and 3
  v += SM_DPP(v, 0x143, 0xc);   // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ u64 wave_scan(u64 v) {
#define SM_ADD(ctrl, rows) v += (u64)(uint32_t)SM_DPP(v >> 32, ctrl, rows) << 32 | (uint32_t)SM_DPP(v, ctrl, rows)
  SM_ADD(0x111, 0xf);
  SM_ADD(0x112, 0xf);
  SM_ADD(0x114, 0xf);
  SM_ADD(0x118, 0xf);
  SM_ADD(0x142, 0xa);
  SM_ADD(0x143, 0xc);
#undef SM_ADD
  return v;
}
__device__ __forceinline__ u64 block_sum(u64 v, Shared& sh) {
  v = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sh.wave_u64[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 s = 0;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += sh.wave_u64[i];
  return s;
}
__device__ __forceinline__ float wave_largest(float v) {   // in lane 63
#define SM_MAX(ctrl, rows) \
  v = fmaxf(v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp((int)0xff800000, (int)__float_as_uint(v), ctrl, rows, 0xf, false)))
  SM_MAX(0x111, 0xf);
  SM_MAX(0x112, 0xf);
  SM_MAX(0x114, 0xf);
  SM_MAX(0x118, 0xf);
  SM_MAX(0x142, 0xa);
  SM_MAX(0x143, 0xc);
#undef SM_MAX
  return v;
}
// (largest a, largest b) over the workgroup
__device__ __forceinline__ void block_max2(float& a, float& b, Shared& sh) {
  a = wave_largest(a);
  b = wave_largest(b);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sh.wave_f[threadIdx.x >> 6] = a, sh.wave_f[16 + (threadIdx.x >> 6)] = b;
  __syncthreads();
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) a = fmaxf(a, sh.wave_f[i]), b = fmaxf(b, sh.wave_f[16 + i]);
}

// ---- bins ------------------------------------------------------------------------------------------------------------------
// Bins of equal width in the logit, bin 0 at the top: monotone, so a bin is a stretch of the walk.
struct BinMap {
  float top, per_unit, last;   // last: the lowest bin, which takes all the rest
  __device__ __forceinline__ float place(float l) const { return (top - l) * per_unit; }   // NaN for infinity under infinity
  __device__ __forceinline__ int bin(float l) const { return l == top ? 0 : (int)fminf(place(l), last); }
};

struct Settings {
  float temp, top_p, min_p, u;
  int top_k;
};
__device__ __forceinline__ Settings settings_of(const SampleArgs& a, int s) {
  Settings o;
  o.temp = a.set.temperature_rows ? a.set.temperature_rows[s] : a.set.temperature;
  o.top_k = a.set.top_k_rows ? a.set.top_k_rows[s] : a.set.top_k;
  o.top_p = a.set.top_p_rows ? a.set.top_p_rows[s] : a.set.top_p;
  o.min_p = a.set.min_p_rows ? a.set.min_p_rows[s] : a.set.min_p;
  o.u = fminf(fmaxf(a.u[(size_t)s * a.u_stride], 0.0f), 1.0f);
  return o;
}
__device__ __forceinline__ u64 nucleus_target(float top_p, u64 S) {   // a mass over this holds top_p of S
  const double want = ceil((double)top_p * (double)S);
  return want < 1.0 ? 0ull : (u64)want - 1ull;
}
__device__ __forceinline__ u64 draw_target(float u, u64 S) {
  const u64 t = (u64)((double)u * (double)S);
  return t < S ? t : S - 1;
}
__device__ __forceinline__ void answer_none(const SampleArgs& a, int b) {
  a.ids[b] = -1;
  if (a.logp) a.logp[b] = -INFINITY;
}
__device__ __forceinline__ void answer(const SampleArgs& a, int b, int id, double w, u64 S) {
  a.ids[b] = id;
  if (a.logp) a.logp[b] = (float)log(w * ONE / (double)S);
}

// ---- sorted lists ----------------------------------------------------------------------------------------------------------
// list[0 .. n) in ascending order; its size is a power of two.  All pairs up to 256 entries, a bitonic network beyond.
__device__ __forceinline__ void sort_places(u64* list, int n, Shared& sh) {
  const int tid = threadIdx.x, nt = blockDim.x;
  if (n <= 256) {
    const int width = n <= 64 ? 64 : n <= 128 ? 128 : 256, e = tid & (width - 1), parts = nt / width, part = tid / width;
    const u64 mine = e < n ? list[e] : 0;
    if (tid < 256) sh.digit_count[tid] = 0;
    __syncthreads();
    if (e < n) {
      uint32_t c = 0;
#pragma unroll 4
      for (int j = part; j < n; j += parts) c += list[j] < mine;
      atomicAdd(&sh.digit_count[e], c);
    }
    __syncthreads();
    if (tid < width && e < n) list[sh.digit_count[e]] = mine;
    __syncthreads();
    return;
  }
  int size = 512;
  while (size < n) size *= 2;
  for (int i = n + tid; i < size; i += nt) list[i] = ~0ull;
  __syncthreads();
#pragma unroll 1
  for (int k = 2; k <= size; k *= 2)
#pragma unroll 1
    for (int j = k / 2; j > 0; j /= 2) {
#pragma unroll 1
      for (int i = tid; i < size / 2; i += nt) {
        const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
        const u64 x = list[lo], y = list[hi];
        if ((x > y) == ((lo & k) == 0)) list[lo] = y, list[hi] = x;
      }
      __syncthreads();
    }
}

// The answer from a sorted list of the row's first n entries of the walk, where nothing after them can be kept (they are all
// there is, or the first top_k).  cum: room for n masses.
__device__ __forceinline__ void draw_from_sorted(const SampleArgs& a, int b, const u64* list, int n, u64* cum, const Scale& sc, const Settings& o, Shared& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, per = (n + blockDim.x - 1) / blockDim.x, e0 = tid * per;
  u64 sum = 0, over = 0;
#pragma unroll 1
  for (int e = e0; e < e0 + per && e < n; ++e) {
    const double w = weight(sc, of_key((uint32_t)(list[e] >> 32)));
    const u64 m = mass_of(w);
    sum += m;
    if (w >= (double)o.min_p) over += m;
    cum[e] = sum;
  }
  u64 base = wave_scan(sum);
  if (lane == 63) sh.wave_u64[wv] = base;
  base -= sum;
  __syncthreads();
  u64 S = 0;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) {
    if (i < wv) base += sh.wave_u64[i];
    S += sh.wave_u64[i];
  }
  // the entry of this thread, if any, at which the mass exceeds t
  auto at_mass = [&](u64 t) SM_INLINE {
    u64 before = base;
    for (int e = e0; e < e0 + per && e < n; ++e) {
      const u64 upto = base + cum[e];
      if (before <= t && t < upto) return e;
      before = upto;
    }
    return -1;
  };
  if (o.top_p < 1.0f) {
    const int e = at_mass(nucleus_target(o.top_p, S));
    if (e >= 0) sh.found_mass = base + cum[e];
    __syncthreads();
    S = sh.found_mass;
  }
  if (o.min_p > 0.0f) {
    over = block_sum(over, sh);
    if (over < S) S = over;
  }
  if (S < ONE_MASS) S = ONE_MASS;   // the largest entry stays whatever is asked
  const int e = at_mass(draw_target(o.u, S));
  if (e >= 0) answer(a, b, (int)(uint32_t)list[e], weight(sc, of_key((uint32_t)(list[e] >> 32))), S);
}

// ---- passes over a row (or a part of one) ----------------------------------------------------------------------------------
// the largest logit and the largest negated one above -inf: this thread's
template <int TYPE> __device__ __forceinline__ void pass_top(const Row<TYPE>& r, float& top, float& low) {
  top = low = -INFINITY;
  r.template each<4>([&](f32x4 k, int) SM_INLINE {
#pragma unroll
    for (int j = 0; j < Row<TYPE>::EPC; ++j) {
      const float l = r.entry(k, j);
      top = fmaxf(top, l);
      low = fmaxf(low, l > -INFINITY ? -l : -INFINITY);
    }
  });
}

// The list of the entries that can be among the k largest of the workgroup's: every thread has its largest one, and the k-th largest
// of those is no larger than the k-th largest of all.  256 bins over them find it; the list takes its bin and those above.
// -> how many, unsorted; more than room: not complete (too many in the last bin, or fewer than k threads have an entry)
template <int LOADS, int TYPE, class I>
__device__ __forceinline__ uint32_t gather_top(const Row<TYPE>& r, int k, float top, float own_max, u64* list, uint32_t room, Shared& sh, I index) {
  const int tid = threadIdx.x, lane = tid & 63, nt = blockDim.x;
  float lowest = own_max > -INFINITY ? -own_max : -INFINITY, unused = 0.0f;
  block_max2(lowest, unused, sh);
  const BinMap map = {top, 255.0f / fmaxf(top + lowest, 1e-30f), 255.0f};
  for (int i = tid; i < 256; i += nt) sh.digit_count[i] = 0;
  if (tid == 0) sh.n = 0, sh.found_bin = 256;
  __syncthreads();
  if (own_max > -INFINITY) atomicAdd(&sh.digit_count[map.bin(own_max)], 1u);
  __syncthreads();
  if (tid < 64) {
    uint32_t c[4], before = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = sh.digit_count[4 * lane + i], before += c[i];
    before = wave_scan(before) - before;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (before < (uint32_t)k && (uint32_t)k <= before + c[i]) sh.found_bin = 4 * lane + i;
      before += c[i];
    }
  }
  __syncthreads();
  const uint32_t cut = sh.found_bin;
  if (cut > 255) return room + 1;
  const float to = cut == 255 ? INFINITY : (float)(cut + 1);
  r.template each_if<LOADS>([&](float l) SM_INLINE { return map.place(l) < to || l == top || to == INFINITY; },
            [&](float l, int i) SM_INLINE {
              const uint32_t at = atomicAdd(&sh.n, 1u);
              if (at < room) list[at] = place_of(l, index(i));
            });
  __syncthreads();
  const uint32_t n = sh.n;
  __syncthreads();
  return n;
}

// bins reach down to 32 temperatures under the top (e^-32 < 2^-45: no mass beyond), or to the lowest logit if that is nearer; the
// largest f32 at most, so that no place is 0 x infinity (what is farther below the top lies in the last bin)
__device__ __forceinline__ BinMap bins_of(const Settings& o, float top, float low, int nbin) {
  return {top, (float)nbin / fmaxf(fminf(fminf(32.0f * o.temp, top + low), 3.4e38f), 1e-30f), (float)(nbin - 1)};
}
__device__ __forceinline__ Scale scale_of(const Settings& o, float top) { return {top, 1.4426950408889634 / (double)o.temp}; }

// masses (and counts, where a rank is asked for) of the bins; -> this thread's mass of the entries with w >= min_p
template <int TYPE>
__device__ __forceinline__ u64 pass_bins(const Row<TYPE>& r, const BinMap& map, const Scale& sc, const Settings& o, bool counted, u64* mass, uint32_t* count) {
  u64 over = 0;
  r.template each<2>([&](f32x4 k, int) SM_INLINE {
#pragma unroll
    for (int j = 0; j < Row<TYPE>::EPC; ++j) {
      const float l = r.entry(k, j);
      if (l > -INFINITY) {
        const double w = weight(sc, l);
        const u64 m = mass_of(w);
        const int bin = map.bin(l);
        if (m) atomicAdd(&mass[bin], m);
        if (counted) atomicAdd(&count[bin], 1u);
        if (w >= (double)o.min_p) over += m;
      }
      if (j & 1) __builtin_amdgcn_sched_barrier(0);   // two entries' registers at a time
    }
  });
  return over;
}

// What several workgroups of a row leave for each other, in the workspace; a row has
//   u64 mass[NSPLIT], over; uint32 count[NSPLIT]; Part part[32]; float cand[parts][KC]; int cand_index[parts][KC];
//   uint32 offset[parts][NSPLIT + 64]; uint16 order[parts][len]: the part's entries by bins, and where a bin of it begins
constexpr int NSPLIT = 4096, KC = 256, MAX_PARTS = 32, OFFSETS = NSPLIT + 64;
constexpr int MAX_LEN = 4 * NSPLIT;   // entries of a part: their order lies where the masses of its bins were, two bytes each
static_assert(MAX_LEN <= 65536 && MAX_LEN * MAX_PARTS >= ST_SAMPLE_MAX_VOCAB, "16-bit order, parts enough");
struct Part {
  float top, low;
  int first;      // index of its first largest entry (greedy rows)
  int complete;   // cand holds its top_k (or all that it has)
};
struct RowSpace {
  u64 *mass, *over;
  uint32_t* count;
  Part* part;
  float* cand;
  int* cand_index;
  uint32_t* offset;
  uint16_t* order;
};
__host__ __device__ inline size_t row_space_bytes(int parts, int len) {   // len: a multiple of 64
  return (size_t)NSPLIT * 12 + 256 + MAX_PARTS * sizeof(Part) + (size_t)parts * (KC * 8 + OFFSETS * 4 + (size_t)len * 2);
}
__device__ __forceinline__ RowSpace row_space(void* ws, int b, int parts, int len) {
  char* p = (char*)ws + (size_t)b * row_space_bytes(parts, len);
  RowSpace s;
  s.mass = (u64*)p, p += (size_t)NSPLIT * 8;
  s.count = (uint32_t*)p, p += (size_t)NSPLIT * 4;
  s.over = (u64*)p, p += 256;
  s.part = (Part*)p, p += MAX_PARTS * sizeof(Part);
  s.cand = (float*)p, p += (size_t)parts * KC * 4;
  s.cand_index = (int*)p, p += (size_t)parts * KC * 4;
  s.offset = (uint32_t*)p, p += (size_t)parts * OFFSETS * 4;
  s.order = (uint16_t*)p;
  return s;
}

// ---- the answer from the bins ----------------------------------------------------------------------------------------------
// list: room for so many places; count may lie at the same address.  SPLIT: the bins' entries are found in the parts' order, not in
// the row.
template <bool SPLIT, int TYPE>
__device__ __forceinline__ void draw_from_bins(const SampleArgs& a, int b, const Row<TYPE>& r, const BinMap& map, const Scale& sc, const Settings& o, bool ranked,
                               u64 over, int nbin, const u64* mass, const uint32_t* count, u64* list, uint32_t room, Shared& sh,
                               const RowSpace& ws, int parts, int len) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, nt = blockDim.x, nw = nt >> 6, per = nbin / nt;
  u64 base_mass = 0;
  uint32_t base_count = 0;
  for (int i = 0; i < per; ++i) {
    base_mass += mass[tid * per + i];
    if (ranked) base_count += count[tid * per + i];
  }
  const u64 own_mass = base_mass;
  const uint32_t own_count = base_count;
  base_mass = wave_scan(base_mass);
  base_count = wave_scan(base_count);
  if (lane == 63) sh.wave_u64[wv] = base_mass, sh.wave_u32[wv] = base_count;
  __syncthreads();
  base_mass -= own_mass;
  base_count -= own_count;
  u64 S = 0;
  uint32_t entries = 0;
  for (int i = 0; i < nw; ++i) {
    if (i < wv) base_mass += sh.wave_u64[i], base_count += sh.wave_u32[i];
    S += sh.wave_u64[i];
    entries += sh.wave_u32[i];
  }
  // three questions, each the entry at which the count or the mass of the walk exceeds a target: the top_k-th entry, the one that
  // completes top_p, the drawn one.  First its bin, then the entry in the bin.
#pragma unroll 1
  for (int question = 0; question < 3; ++question) {
    const bool by_count = question == 0;
    u64 target;
    if (question == 0) {
      if (!ranked || (uint32_t)o.top_k >= entries) continue;
      target = (u64)(o.top_k - 1);
    } else if (question == 1) {
      if (!(o.top_p < 1.0f)) continue;
      target = nucleus_target(o.top_p, S);
    } else {
      if (o.min_p > 0.0f && over < S) S = over;
      if (S < ONE_MASS) S = ONE_MASS;   // the largest entry stays whatever is asked
      target = draw_target(o.u, S);
    }
    if (tid == 0) sh.n = 0, sh.found_bin = 0, sh.found_count = 0, sh.found_mass = 0, sh.found_place = 0;
    __syncthreads();
    {
      u64 m0 = base_mass;
      uint32_t c0 = base_count;
#pragma unroll 1
      for (int i = 0; i < per; ++i) {
        const u64 m1 = m0 + mass[tid * per + i];
        const uint32_t c1 = by_count ? c0 + count[tid * per + i] : 0;
        if (by_count ? c0 <= target && target < c1 : m0 <= target && target < m1) sh.found_bin = tid * per + i, sh.found_count = c0, sh.found_mass = m0;
        m0 = m1;
        c0 = c1;
      }
    }
    __syncthreads();
    const int bin = (int)sh.found_bin;
    u64 before_mass = sh.found_mass;
    uint32_t before_count = by_count ? sh.found_count : 0;
    // the bin's entries: one list (the counts are not needed any more once the first question has its bin)
    const float from = (float)bin, to = bin == nbin - 1 ? INFINITY : (float)(bin + 1);
    auto in_bin = [&](float l) SM_INLINE {
      const float at = map.place(l);
      return (at >= from && (at < to || to == INFINITY)) || (bin == 0 && l == map.top);
    };
    auto element = [&](uint32_t t) SM_INLINE {   // SPLIT: the place of the bin's t-th entry
      int g = 0;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) g += sh.part_end[g + d - 1] <= t ? d : 0;
      const int i = g * len + ws.order[(size_t)g * len + (uint32_t)(sh.part_at[g] + t)];   // (the sum, modulo 2^32, is the place in the part)
      return place_of(logit<TYPE>(r.p[min(i, r.n - 1)]), i);
    };
    if constexpr (SPLIT) {
      if (wv == 0) {
        uint32_t from_at = 0, n = 0;
        if (lane < parts) {
          from_at = ws.offset[(size_t)lane * OFFSETS + bin];
          n = ws.offset[(size_t)lane * OFFSETS + bin + 1] - from_at;
        }
        const uint32_t end = wave_scan(n);
        if (lane < MAX_PARTS) sh.part_end[lane] = end, sh.part_at[lane] = from_at - (end - n);
        if (lane == 63) sh.n = end;
      }
      __syncthreads();
      if (sh.n <= room)
        for (uint32_t t = tid; t < sh.n; t += nt) list[t] = element(t);
    } else {
      r.template each_if<4>(in_bin, [&](float l, int i) SM_INLINE {
        const uint32_t at = atomicAdd(&sh.n, 1u);
        if (at < room) list[at] = place_of(l, i);
      });
    }
    __syncthreads();
    const uint32_t n_bin = sh.n;
    __syncthreads();
    // More of the row in one bin than the list holds (equal logits, mostly): the rounds below go over the row itself, twice a round, and
    // that takes its time.  us, as in text / three values / one value: 4096 x 9339 top_p 0.9 150 / 665 / 815, with top_k 50 57 / 1057 /
    // 1372; 1 x 131072 24 / 376 / 1051, 27 / 568 / 1665.
    const bool from_row = n_bin > room;
    auto walk = [&](auto f) SM_INLINE {   // f(place) for this thread's share of the bin
      if (SPLIT || !from_row) {
#pragma unroll 1
        for (uint32_t i = tid; i < n_bin; i += nt) f(SPLIT && from_row ? element(i) : list[i]);
      } else if constexpr (!SPLIT) {
        r.template each_if<4>(in_bin, [&](float l, int i) SM_INLINE { f(place_of(l, i)); });
      }
    };
    // eight bits of the place a round, from the highest one in which two elements differ, until one wave can compare the rest
    u64 prefix = 0;
    int high = 64;   // the bits from `high` on are settled: prefix's
#pragma unroll 1
    for (int round = 0; round < 9; ++round) {   // the ninth has 64 bits settled
      auto inside = [&](u64 place) SM_INLINE { return high >= 64 || (place >> high) == (prefix >> high); };
      uint32_t n = n_bin;
      int top_bit = 64;
      if (n_bin > 64 || from_row) {
        u64 any = 0, every = ~0ull;
        n = 0;
        walk([&](u64 place) SM_INLINE {
          if (inside(place)) any |= place, every &= place, ++n;
        });
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) any |= __shfl_xor(any, d, 64), every &= __shfl_xor(every, d, 64), n += __shfl_xor(n, d, 64);
        __syncthreads();
        if (lane == 0) sh.wave_any[wv] = any, sh.wave_all[wv] = every, sh.wave_u32[wv] = n;
        for (int i = tid; i < 256; i += nt) sh.digit_mass[i] = 0, sh.digit_count[i] = 0;
        __syncthreads();
        any = 0, every = ~0ull, n = 0;
        for (int i = 0; i < nw; ++i) any |= sh.wave_any[i], every &= sh.wave_all[i], n += sh.wave_u32[i];
        top_bit = 64 - __clzll(any ^ every);   // above the highest bit that differs (two places are never equal)
        prefix = top_bit >= 64 ? 0 : (any >> top_bit) << top_bit;
      }
      const bool few = n <= 64;
      if (tid == 0) sh.n = 0;
      if (few && tid < 64) sh.digit_count[tid] = 0, sh.digit_mass[128 + tid] = 0;
      __syncthreads();
      const int low_bit = top_bit > 8 ? top_bit - 8 : 0;
      // few: the digits' array takes the elements themselves, and their masses behind them
      walk([&](u64 place) SM_INLINE {
        if (!inside(place)) return;
        const u64 m = mass_of(weight(sc, of_key((uint32_t)(place >> 32))));
        if (few) {
          const uint32_t at = atomicAdd(&sh.n, 1u);
          sh.digit_mass[at] = place;
          sh.digit_mass[64 + at] = m;
        } else {
          const int d = (int)(place >> low_bit) & 255;
          if (by_count) atomicAdd(&sh.digit_count[d], 1u);
          atomicAdd(&sh.digit_mass[d], m);
        }
      });
      __syncthreads();
      if (few) {
        // every element against every other: each wave takes its share of the others
        const u64 mine = lane < (int)n ? sh.digit_mass[lane] : 0;
        uint32_t c = 0;
        u64 mb = 0;
        for (int i = wv; i < (int)n; i += nw)
          if (sh.digit_mass[i] < mine) ++c, mb += sh.digit_mass[64 + i];
        if (c) {
          atomicAdd(&sh.digit_count[lane], c);
          atomicAdd(&sh.digit_mass[128 + lane], mb);
        }
        __syncthreads();
        if (wv == 0 && lane < (int)n) {
          const u64 m = sh.digit_mass[64 + lane];
          c = before_count + sh.digit_count[lane];
          mb = before_mass + sh.digit_mass[128 + lane];
          if (by_count ? c == target : mb <= target && target < mb + m) sh.found_place = mine, sh.found_mass = mb + m;
        }
        __syncthreads();
        break;
      }
      if (wv == 0) {
        uint32_t c[4], ct = 0;
        u64 m[4], mt = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = sh.digit_count[4 * lane + i], m[i] = sh.digit_mass[4 * lane + i], ct += c[i], mt += m[i];
        ct = before_count + wave_scan(ct) - ct;
        mt = before_mass + wave_scan(mt) - mt;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (by_count ? ct <= target && target < ct + c[i] : mt <= target && target < mt + m[i]) sh.found_bin = 4 * lane + i, sh.found_count = ct, sh.found_mass = mt;
          ct += c[i];
          mt += m[i];
        }
      }
      __syncthreads();
      prefix |= (u64)(sh.found_bin & 255) << low_bit;
      high = low_bit;
      before_count = sh.found_count;
      before_mass = sh.found_mass;
    }
    if (question < 2) S = sh.found_mass;
    __syncthreads();
  }
  if (tid == 0) answer(a, b, (int)(uint32_t)sh.found_place, weight(sc, of_key((uint32_t)(sh.found_place >> 32))), S);
}

// ---- kernels ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ bool is_greedy(const Settings& o) { return !(o.temp > 0.0f) || o.top_k == 1; }
// a list of the top_k can be had from the threads' largest entries, twice as many as are asked for
__device__ __forceinline__ bool by_list(const Settings& o, int chunks) { return o.top_k > 0 && o.top_k <= min(min((int)blockDim.x, chunks) / 2, KC); }

// One workgroup a row.  Dynamic shared memory: masses of the bins [nbin], a list of places [nbin / 2] (before that, counts).
// LISTS: rows that a sorted list answers (greedy ones, short ones, a top_k that the threads' largest entries bound); BINS: any row.
// With LISTS alone a row that needs the bins is marked TODO in ids, and BINS alone takes the marked ones (todo) or all.  Apart, the
// lists' kernel needs 64 registers and the chip holds twice as many rows of it: 4096 x 9339 with top-k 79 us together, 59 apart.
constexpr int TODO = -2;
template <int TYPE, bool LISTS, bool BINS, int WAVES>
__global__ __launch_bounds__(BINS ? 1024 : 512, WAVES) void sample_row_kernel(SampleArgs a, int nbin, int todo) {
  typedef typename LOf<TYPE>::t T;
  extern __shared__ __align__(16) char dyn[];
  __shared__ Shared sh;
  const int b = blockIdx.x, tid = threadIdx.x, nt = blockDim.x;
  if (a.n_dev && a.row0 + b >= *a.n_dev) return;
  if (todo && a.ids[b] != TODO) return;
  u64* const mass = (u64*)dyn;
  u64* const list = mass + nbin;
  uint32_t* const count = (uint32_t*)list;
  const uint32_t room = nbin / 2;
  const Settings o = settings_of(a, a.idx ? a.idx[b] : b);
  const Row<TYPE> r((const T*)a.logits + (size_t)b * a.ld, a.V);
  float top, low;
  pass_top(r, top, low);
  const float own_max = top;
  block_max2(top, low, sh);
  if (top == -INFINITY) {
    if (tid == 0) answer_none(a, b);
    return;
  }
  const Scale sc = scale_of(o, top);
  if constexpr (LISTS) {
    if (is_greedy(o)) {
      if (tid == 0) sh.n = 0xffffffffu;
      __syncthreads();
      r.template each_if<4>([&](float l) SM_INLINE { return l == top; }, [&](float, int i) SM_INLINE { atomicMin(&sh.n, (uint32_t)i); });
      __syncthreads();
      if (tid == 0) answer(a, b, (int)sh.n, 1.0, ONE_MASS);
      return;
    }
    const bool listed = by_list(o, r.chunks);
    if (listed || a.V <= (int)room) {
      uint32_t n = room + 1;
      if (listed && a.V > 256) n = gather_top<4>(r, o.top_k, top, own_max, list, room, sh, [](int i) SM_INLINE { return i; });
      if (n > room && a.V <= (int)room) {   // all entries, where they fit: also those of a row with fewer than top_k threads that have one
        if (tid == 0) sh.n = 0;
        __syncthreads();
        r.template each_if<2>([](float l) SM_INLINE { return l > -INFINITY; }, [&](float l, int i) SM_INLINE {
          const uint32_t at = atomicAdd(&sh.n, 1u);
          if (at < room) list[at] = place_of(l, i);
        });
        __syncthreads();
        n = sh.n;
        __syncthreads();
      }
      if (n <= room) {
        sort_places(list, (int)n, sh);
        draw_from_sorted(a, b, list, o.top_k > 0 ? min((int)n, o.top_k) : (int)n, mass, sc, o, sh);
        return;
      }
    }
    if constexpr (!BINS) {
      if (tid == 0) a.ids[b] = TODO;
      return;
    }
  }
  if constexpr (BINS) {
    const BinMap map = bins_of(o, top, low, nbin);
    const bool ranked = o.top_k > 0 && o.top_k < a.V;
    for (int i = tid; i < nbin; i += nt) {
      mass[i] = 0;
      if (ranked) count[i] = 0;
    }
    __syncthreads();
    u64 over = pass_bins(r, map, sc, o, ranked, mass, count);
    __syncthreads();
    if (o.min_p > 0.0f) over = block_sum(over, sh);
    draw_from_bins<false>(a, b, r, map, sc, o, ranked, over, nbin, mass, count, list, room, sh, RowSpace{}, 0, 0);
  }
}

// A long row over several workgroups, in three launches: (1) every part's largest entry, and its top_k where a list of them will do;
// (2) masses of the bins, added up in the workspace (whole numbers: in any order the same); (3) one workgroup a row draws.
template <int TYPE> __global__ __launch_bounds__(512) void sample_part_kernel(SampleArgs a, int parts, int len) {
  typedef typename LOf<TYPE>::t T;
  __shared__ Shared sh;
  __shared__ u64 list[1024];
  const int b = blockIdx.y, g = blockIdx.x, tid = threadIdx.x, nt = blockDim.x;
  if (a.n_dev && a.row0 + b >= *a.n_dev) return;
  const RowSpace ws = row_space(a.ws, b, parts, len);
  for (int i = g * nt + tid; i < NSPLIT; i += parts * nt) ws.mass[i] = 0, ws.count[i] = 0;
  if (g == 0 && tid == 0) *ws.over = 0;
  const Settings o = settings_of(a, a.idx ? a.idx[b] : b);
  const int i0 = g * len;
  const Row<TYPE> r((const T*)a.logits + (size_t)b * a.ld + i0, min(len, a.V - i0));
  float top, low;
  pass_top(r, top, low);
  const float own_max = top;
  block_max2(top, low, sh);
  int complete = 1;
  if (tid == 0) sh.n = 0xffffffffu;
  __syncthreads();
  if (top > -INFINITY && is_greedy(o)) {
    r.template each_if<4>([&](float l) SM_INLINE { return l == top; }, [&](float, int i) SM_INLINE { atomicMin(&sh.n, (uint32_t)(i0 + i)); });
    __syncthreads();
  } else if (by_list(o, 1024)) {
    uint32_t n = 0;
    if (top > -INFINITY) n = gather_top<4>(r, o.top_k, top, own_max, list, 1024, sh, [&](int i) SM_INLINE { return i0 + i; });
    complete = n <= 1024;
    if (complete) {
      if (n > (uint32_t)o.top_k) sort_places(list, (int)n, sh);
      for (int i = tid; i < KC; i += nt) {
        const bool in = i < (int)n && i < o.top_k;
        ws.cand[g * KC + i] = in ? of_key((uint32_t)(list[i] >> 32)) : -INFINITY;
        ws.cand_index[g * KC + i] = in ? (int)(uint32_t)list[i] : 0;
      }
    }
  }
  if (tid == 0) ws.part[g] = {top, low, (int)sh.n, complete};
}

// what all parts of a row have together, a lane a part (every wave for itself)
__device__ __forceinline__ void join_parts(const RowSpace& ws, int parts, float& top, float& low, bool& complete, int& first) {
  const int lane = threadIdx.x & 63;
  Part p = {-INFINITY, -INFINITY, -1, 1};
  if (lane < parts) p = ws.part[lane];
  top = __shfl(wave_largest(p.top), 63, 64);
  low = __shfl(wave_largest(p.low), 63, 64);
  complete = __ballot(!p.complete) == 0;
  first = __shfl(p.first, __ffsll(__ballot(p.top == top)) - 1, 64);   // of the first part with the largest
}

template <int TYPE> __global__ __launch_bounds__(512) void sample_bins_kernel(SampleArgs a, int parts, int len) {
  typedef typename LOf<TYPE>::t T;
  extern __shared__ __align__(16) char dyn[];
  __shared__ Shared sh;
  const int b = blockIdx.y, g = blockIdx.x, tid = threadIdx.x, nt = blockDim.x;
  if (a.n_dev && a.row0 + b >= *a.n_dev) return;
  const RowSpace ws = row_space(a.ws, b, parts, len);
  const Settings o = settings_of(a, a.idx ? a.idx[b] : b);
  float top, low;
  bool complete;
  int first;
  join_parts(ws, parts, top, low, complete, first);
  if (top == -INFINITY || is_greedy(o) || (by_list(o, 1024) && complete)) return;   // no bins are needed
  const int i0 = g * len;
  const Row<TYPE> r((const T*)a.logits + (size_t)b * a.ld + i0, min(len, a.V - i0));
  u64* const mass = (u64*)dyn;
  uint32_t* const count = (uint32_t*)(mass + NSPLIT);
  const bool ranked = o.top_k > 0 && o.top_k < a.V;
  for (int i = tid; i < NSPLIT; i += nt) mass[i] = 0, count[i] = 0;
  __syncthreads();
  const BinMap map = bins_of(o, top, low, NSPLIT);
  u64 over = pass_bins(r, map, scale_of(o, top), o, true, mass, count);
  if (o.min_p > 0.0f) {
    over = block_sum(over, sh);
    if (tid == 0 && over) atomicAdd(ws.over, over);
  }
  __syncthreads();
  for (int i = tid; i < NSPLIT; i += nt) {
    if (mass[i]) atomicAdd(&ws.mass[i], mass[i]);
    if (ranked && count[i]) atomicAdd(&ws.count[i], count[i]);
  }
  // the entries by bins, so that the last kernel need not look for them: where each bin begins, and then every entry in its place
  constexpr int PER = NSPLIT / 512;
  uint32_t c[PER], before = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) c[i] = count[tid * PER + i], before += c[i];
  const uint32_t own = before;
  before = wave_scan(before);
  if ((tid & 63) == 63) sh.wave_u32[tid >> 6] = before;
  __syncthreads();   // and nobody reads the counts any more
  before -= own;
  for (int i = 0; i < (tid >> 6); ++i) before += sh.wave_u32[i];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    count[tid * PER + i] = before;
    ws.offset[(size_t)g * OFFSETS + tid * PER + i] = before;
    before += c[i];
  }
  if (tid == nt - 1) ws.offset[(size_t)g * OFFSETS + NSPLIT] = before;
  __syncthreads();
  uint16_t* const order = (uint16_t*)mass;
  r.template each<4>([&](f32x4 k, int ch) SM_INLINE {
#pragma unroll
    for (int j = 0; j < Row<TYPE>::EPC; ++j) {
      const float l = r.entry(k, j);
      if (l > -INFINITY) {
        const uint32_t at = atomicAdd(&count[map.bin(l)], 1u);
        if (at < (uint32_t)len) order[at] = (uint16_t)(ch * Row<TYPE>::EPC + j - r.pad);
      }
    }
  });
  __syncthreads();
  // (places that no entry has are copied too, and never read)
  for (int i = tid; i < len / 4; i += nt) ((u64*)(ws.order + (size_t)g * len))[i] = mass[i];
}

constexpr int JOIN_ROOM = MAX_PARTS * KC;   // places in the list: all parts' candidates
template <int TYPE> __global__ __launch_bounds__(1024) void sample_join_kernel(SampleArgs a, int parts, int len) {
  typedef typename LOf<TYPE>::t T;
  extern __shared__ __align__(16) char dyn[];
  __shared__ Shared sh;
  const int b = blockIdx.x, tid = threadIdx.x, nt = blockDim.x;
  if (a.n_dev && a.row0 + b >= *a.n_dev) return;
  const RowSpace ws = row_space(a.ws, b, parts, len);
  const Settings o = settings_of(a, a.idx ? a.idx[b] : b);
  u64* const mass = (u64*)dyn;
  u64* const list = mass + NSPLIT;
  uint32_t* const count = (uint32_t*)list;
  const uint32_t room = JOIN_ROOM;
  float top, low;
  bool complete;
  int first;
  join_parts(ws, parts, top, low, complete, first);
  if (top == -INFINITY || is_greedy(o)) {
    if (tid == 0) {
      if (top == -INFINITY) answer_none(a, b);
      else answer(a, b, first, 1.0, ONE_MASS);
    }
    return;
  }
  const Scale sc = scale_of(o, top);
  const Row<TYPE> r((const T*)a.logits + (size_t)b * a.ld, a.V);
  const BinMap map = bins_of(o, top, low, NSPLIT);
  const bool ranked = o.top_k > 0 && o.top_k < a.V;
  // (half of the part kernel's threads: what it took for a list is one here)
  if (o.top_k > 0 && o.top_k <= KC && complete) {
    const Row<ST_TYPE_F32> c(ws.cand, parts * KC);
    float own, unused;
    pass_top(c, own, unused);
    uint32_t n = gather_top<4>(c, o.top_k, top, own, list, room, sh, [&](int i) SM_INLINE { return ws.cand_index[i]; });
    if (n > room) {   // too few threads have one: all of them, JOIN_ROOM at most
      if (tid == 0) sh.n = 0;
      __syncthreads();
      for (int i = tid; i < parts * KC; i += nt)
        if (ws.cand[i] > -INFINITY) list[atomicAdd(&sh.n, 1u)] = place_of(ws.cand[i], ws.cand_index[i]);
      __syncthreads();
      n = sh.n;
      __syncthreads();
    }
    sort_places(list, (int)n, sh);
    draw_from_sorted(a, b, list, min((int)n, o.top_k), mass, sc, o, sh);
    return;
  }
  for (int i = tid; i < NSPLIT; i += nt) {
    mass[i] = ws.mass[i];
    if (ranked) count[i] = ws.count[i];
  }
  const u64 over = *ws.over;
  __syncthreads();
  draw_from_bins<true>(a, b, r, map, sc, o, ranked, over, NSPLIT, mass, count, list, room, sh, ws, parts, len);
}

// Parts of a row: few long rows leave most of the chip idle, and one workgroup takes its time over a long row.  About two workgroups
// a CU, parts of 4096 entries and more (and MAX_LEN at most); for fewer than four the three launches do not pay.
int parts_of(int B, int V, int* len) {
  int g = V < 16384 ? 1 : 512 / B;
  if (g < 4) return 1;
  if (g > V / 4096) g = V / 4096;
  if (g < (V + MAX_LEN - 1) / MAX_LEN) g = (V + MAX_LEN - 1) / MAX_LEN;
  if (g > MAX_PARTS) g = MAX_PARTS;
  *len = ((V + g - 1) / g + 63) / 64 * 64;
  return (V + *len - 1) / *len;   // those that have entries
}

template <int TYPE> int launch_type(const SampleArgs& a, hipStream_t st) {
  int len = 0;
  const int parts = parts_of(a.B, a.V, &len);
  if (parts == 1) {
    // Bins, and half as many places in the list.  Up to 1024 entries the list takes any row, so that no row is marked and one launch is
    // enough: with 1024 / 2048 bins 4096 x 777 settings by row 31.6 / 28.4 us, 600 x 777 top_k 50 10.8 / 9.2; unfiltered draws pay for
    // it, they sort the list where bins would do: 4096 x 777 40 / 99 us, 1 x 777 8.9 / 23.  Beyond, with 1024 / 2048 / 4096 bins, us:
    // 128 x 9339 15.3 / 15.3 / 16.3, 1024 x 9339 top_k 400 42.9 / 44.0 / 48.5; 1024 x 19724 62.7 / 59.6 / 61.1, top_p 0.9 73.5 / 71.4 /
    // 73.4, top_k 400 70.4 / 71.4 / 74.9; 200 x 50001 top_k 400 45.2 / 45.3 / 46.2, unfiltered 46.8 / 45.9 / 39.4; 256 x 131072 190 /
    // 104 / 103, top_p 0.9 126 / 122 / 117.
    const int nbin = a.V <= 1024 ? 2048 : a.V <= 16384 ? 1024 : a.V <= 65536 ? 2048 : 4096;
    const size_t lds = (size_t)nbin * 12;
    // 256 x 131072 bf16: 151 us with 1024, 189 with 512; 128 x 9339: 16.0 and 14.5
    const int threads = a.V <= 2048 ? 256 : a.V <= 32768 ? 512 : 1024;
    const bool alike = !a.set.temperature_rows && !a.set.top_k_rows;
    const bool lists = a.V <= nbin / 2 || (alike && (!(a.set.temperature > 0.0f) || (a.set.top_k > 0 && a.set.top_k <= 128)));
    const long rows = ((1L << 32) - 1) / threads;   // a launch has fewer than 2^32 threads
    ST_CHECK_ARG(a.B <= rows, "B=%d: at most %ld rows of %d values in one call", a.B, rows, a.V);
    // Lists by a kernel of their own / by the one that has both, top_k 50, us.  9339 entries: 64 rows 13.1 / 9.6, 512 rows 14.1 / 11.9,
    // 1024 rows 20.6 / 22.0, 4096 rows 56.8 / 74.8; 3000: 512 rows 10.8 / 9.9, 1024 rows 13.0 / 16.7; 50001: 256 rows 31.8 / 23.5, 512
    // rows 38.9 / 41.4.  (With settings by row, longer rows than the list take the kernel that has both: 4096 x 9339 76 us where one
    // setting for all takes 57.)
    if (lists && a.B >= 512) {
      hipLaunchKernelGGL((sample_row_kernel<TYPE, true, false, 8>), dim3(a.B), dim3(256), lds, st, a, nbin, 0);
      ST_LAUNCH_CHECK();
      // rows marked: their equal logits did not fit into a list, or too few threads had an entry (a list of nbin / 2 takes any shorter row)
      if (a.V > nbin / 2 && a.set.top_k != 1 && a.set.temperature > 0.0f)
        hipLaunchKernelGGL((sample_row_kernel<TYPE, false, true, 4>), dim3(a.B), dim3(threads), lds, st, a, nbin, 1);
    } else if (alike && !lists) {
      hipLaunchKernelGGL((sample_row_kernel<TYPE, false, true, 4>), dim3(a.B), dim3(threads), lds, st, a, nbin, 0);
    } else {
      hipLaunchKernelGGL((sample_row_kernel<TYPE, true, true, 4>), dim3(a.B), dim3(threads), lds, st, a, nbin, 0);
    }
    ST_LAUNCH_CHECK();
    return ST_OK;
  }
  ST_CHECK_ARG(parts <= MAX_PARTS && len <= MAX_LEN, "V=%d in %d parts of %d", a.V, parts, len);
  constexpr int join_lds = NSPLIT * 8 + JOIN_ROOM * 8;
  ST_ENSURE_LDS(sample_join_kernel<TYPE>, join_lds);
  hipLaunchKernelGGL((sample_part_kernel<TYPE>), dim3(parts, a.B), dim3(512), 0, st, a, parts, len);
  ST_LAUNCH_CHECK();
  hipLaunchKernelGGL((sample_bins_kernel<TYPE>), dim3(parts, a.B), dim3(512), (size_t)NSPLIT * 12, st, a, parts, len);
  ST_LAUNCH_CHECK();
  hipLaunchKernelGGL((sample_join_kernel<TYPE>), dim3(a.B), dim3(1024), join_lds, st, a, parts, len);
  ST_LAUNCH_CHECK();
  return ST_OK;
}

}  // namespace

// the most that a call with up to B rows needs (fewer rows are cut into more parts)
size_t sample_workspace_most(int B, int V) {
  size_t most = 0;
  for (int n = B < 128 ? B : 128; n > 0; --n) most = sample_workspace(n, V) > most ? sample_workspace(n, V) : most;   // 128: parts_of's 4 parts
  return most;
}
size_t sample_workspace(int B, int V) {
  int len = 0;
  const int parts = parts_of(B, V, &len);
  return parts == 1 ? 0 : (size_t)B * row_space_bytes(parts, len);
}

int sample_launch(const SampleArgs& a, hipStream_t st) {
  return a.type == ST_TYPE_F32 ? launch_type<ST_TYPE_F32>(a, st) : a.type == ST_TYPE_BF16 ? launch_type<ST_TYPE_BF16>(a, st) : launch_type<ST_TYPE_F16>(a, st);
}

int sample_check(const StSampleSettings* s) {
  ST_CHECK_ARG(s != nullptr, "settings struct is NULL");
  ST_CHECK_ARG(s->temperature_rows || (s->temperature >= 0.0f && s->temperature < INFINITY), "temperature=%g must be finite and not negative", s->temperature);
  ST_CHECK_ARG(s->top_k_rows || s->top_k >= 0, "top_k=%d must not be negative (0: off)", s->top_k);
  ST_CHECK_ARG(s->top_p_rows || (s->top_p > 0.0f && s->top_p <= 1.0f), "top_p=%g must lie in (0, 1]", s->top_p);
  ST_CHECK_ARG(s->min_p_rows || (s->min_p >= 0.0f && s->min_p <= 1.0f), "min_p=%g must lie in [0, 1]", s->min_p);
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
  ST_CHECK_ARG(((size_t)workspace & 15) == 0, "the workspace must lie on 16 bytes");
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
