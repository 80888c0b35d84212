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
template <int TYPE> __device__ __forceinline__ typename LOf<TYPE>::t no_entry() {
  if constexpr (TYPE == ST_TYPE_BF16) return 0xff80;
  else return (typename LOf<TYPE>::t)-INFINITY;
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
// 16-byte chunks on the row's own alignment: chunk c holds the entries c * EPC - pad + 0..EPC-1, of which those outside the row
// read as no entry.  Either in global memory, where only a chunk that lies in the row is loaded at once, or copied to shared memory.
template <int TYPE> struct Chunk {
  typedef typename LOf<TYPE>::t T;
  static constexpr int EPC = 16 / sizeof(T);
  T v[EPC];
};
template <int TYPE> struct Row {
  typedef typename LOf<TYPE>::t T;
  static constexpr int EPC = Chunk<TYPE>::EPC;
  const T* p;          // entry 0
  const void* local;   // shared memory, or null
  int n, pad, chunks;
  __device__ Row(const T* p_, int n_) : p(p_), local(nullptr), n(n_) {
    pad = (int)(((size_t)p & 15) / sizeof(T));
    chunks = (n + pad + EPC - 1) / EPC;
  }
  __device__ __forceinline__ Chunk<TYPE> global(int c) const {
    Chunk<TYPE> k;
    const int i0 = c * EPC - pad;
    if (i0 >= 0 && i0 + EPC <= n) {
      *(f32x4*)k.v = *(const f32x4*)(p + i0);
    } else {
#pragma unroll
      for (int j = 0; j < EPC; ++j) k.v[j] = i0 + j >= 0 && i0 + j < n ? p[i0 + j] : no_entry<TYPE>();
    }
    return k;
  }
  template <bool LOCAL> __device__ __forceinline__ Chunk<TYPE> chunk(int c) const {
    if constexpr (LOCAL) {
      Chunk<TYPE> k;
      *(f32x4*)k.v = ((const f32x4*)local)[c];
      return k;
    } else {
      return global(c);
    }
  }
};
// f(logit, index) for this thread's share of the entries above -inf
template <int TYPE, bool LOCAL, class F> __device__ __forceinline__ void each_entry(const Row<TYPE>& r, F f) {
  constexpr int EPC = Row<TYPE>::EPC;
#pragma unroll 2
  for (int c = threadIdx.x; c < r.chunks; c += blockDim.x) {
    const Chunk<TYPE> k = r.template chunk<LOCAL>(c);
#pragma unroll
    for (int j = 0; j < EPC; ++j) {
      const float l = logit<TYPE>(k.v[j]);
      if (l > -INFINITY) f(l, c * EPC + j - r.pad);
    }
  }
}

// ---- sums over the workgroup ---------------------------------------------------------------------------------------------
struct Shared {
  u64 digit_mass[256];
  uint32_t digit_count[256];
  u64 small[64];
  u64 wave_u64[16];
  uint32_t wave_u32[16];
  float wave_f[32];
  u64 found_place, found_mass;
  uint32_t found_count, found_bin, n;
};

// one wave's choice among n <= 64 elements (lane i: `place`, `m`; elements of shared memory at places[] and masses[])
template <bool BY_COUNT>
__device__ __forceinline__ void pick_of_64(Shared& sh, const u64* places, const u64* masses, int n, u64 target, u64 before_mass, uint32_t before_count) {
  const int lane = threadIdx.x & 63;
  const u64 mine = lane < n ? places[lane] : ~0ull, m = lane < n ? masses[lane] : 0;
  uint32_t c = before_count;
  u64 b = before_mass;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const bool earlier = places[i] < mine;
    c += earlier;
    b += earlier ? masses[i] : 0;
  }
  const bool here = lane < n && (BY_COUNT ? c == target : b <= target && target < b + m);
  if (here) sh.found_place = mine, sh.found_count = c, sh.found_mass = b;
}

__device__ __forceinline__ u64 wave_scan(u64 v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ u64 block_sum(u64 v, Shared& sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.wave_u64[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 s = 0;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += sh.wave_u64[i];
  return s;
}
// (largest a, largest b) over the workgroup
__device__ __forceinline__ void block_max2(float& a, float& b, Shared& sh) {
  a = wave_max(a);
  b = wave_max(b);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.wave_f[threadIdx.x >> 6] = a, sh.wave_f[16 + (threadIdx.x >> 6)] = b;
  __syncthreads();
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) a = fmaxf(a, sh.wave_f[i]), b = fmaxf(b, sh.wave_f[16 + i]);
}

// ---- the entry at which a sum passes its target ----------------------------------------------------------------------------
// Among the elements that `each` gives (f(place, mass)), walked in the order of their places: the first at which the count (or the
// mass) walked so far, it included, exceeds `target`.  sh.found_*: its place, and count and mass before it.  Eight bits of the
// place a round, from the highest one in which two elements differ, until 64 elements are left for one wave.
template <bool BY_COUNT, class E> __device__ void select(Shared& sh, u64 target, E each) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  u64 prefix = 0, before_mass = 0;
  uint32_t before_count = 0;
  int low = 64;   // the bits from `low` on are settled and equal to prefix's
  for (;;) {
    auto inside = [&](u64 place) { return low >= 64 || (place >> low) == (prefix >> low); };
    // how many are left, and where they differ
    u64 any = 0, all = ~0ull;
    uint32_t n = 0;
    each([&](u64 place, u64) {
      if (inside(place)) any |= place, all &= place, ++n;
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) any |= __shfl_xor(any, o, 64), all &= __shfl_xor(all, o, 64), n += __shfl_xor(n, o, 64);
    __syncthreads();
    if (tid == 0) sh.n = 0;
    if (lane == 0) sh.wave_u64[wv] = any, sh.digit_mass[wv] = all, sh.wave_u32[wv] = n;
    __syncthreads();
    any = 0, all = ~0ull, n = 0;
    for (int i = 0; i < (int)(blockDim.x >> 6); ++i) any |= sh.wave_u64[i], all &= sh.digit_mass[i], n += sh.wave_u32[i];
    __syncthreads();
    if (n <= 64) {
      each([&](u64 place, u64 m) {
        if (inside(place)) {
          const uint32_t at = atomicAdd(&sh.n, 1u);
          sh.small[at] = place;
          sh.digit_mass[at] = m;
        }
      });
      __syncthreads();
      if (wv == 0) pick_of_64<BY_COUNT>(sh, sh.small, sh.digit_mass, (int)n, target, before_mass, before_count);
      __syncthreads();
      return;
    }
    const int high = 64 - __clzll(any ^ all);   // above the highest bit that differs; two places are never equal
    low = high > 8 ? high - 8 : 0;
    prefix = high >= 64 ? 0 : (any >> high) << high;
    auto within = [&](u64 place) { return high >= 64 || (place >> high) == (prefix >> high); };
    for (int i = tid; i < 256; i += blockDim.x) sh.digit_mass[i] = 0, sh.digit_count[i] = 0;
    __syncthreads();
    each([&](u64 place, u64 m) {
      if (within(place)) {
        const int d = (int)(place >> low) & 255;
        if constexpr (BY_COUNT) atomicAdd(&sh.digit_count[d], 1u);
        atomicAdd(&sh.digit_mass[d], m);
      }
    });
    __syncthreads();
    if (wv == 0) {
      uint32_t c[4], ct = 0;
      u64 m[4], mt = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = sh.digit_count[4 * lane + i], m[i] = sh.digit_mass[4 * lane + i], ct += c[i], mt += m[i];
      ct = before_count + wave_scan(ct, lane) - ct;
      mt = before_mass + wave_scan(mt, lane) - mt;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool here = BY_COUNT ? ct <= target && target < (u64)ct + c[i] : mt <= target && target < mt + m[i];
        if (here) sh.found_bin = 4 * lane + i, sh.found_count = ct, sh.found_mass = mt;
        ct += c[i];
        mt += m[i];
      }
    }
    __syncthreads();
    prefix |= (u64)sh.found_bin << low;
    before_count = sh.found_count;
    before_mass = sh.found_mass;
  }
}

// ---- bins ------------------------------------------------------------------------------------------------------------------
// Bins of equal width in the logit, bin 0 at the top: monotone, so a bin is a stretch of the walk.
struct Bins {
  u64* mass;           // [n]
  uint32_t* count;     // [n], where the list lies later
  u64* list;           // [n / 2] places
  int n;
  float top, per_unit;
};
__device__ __forceinline__ int bin_of(const Bins& b, float l) {
  return l == b.top ? 0 : (int)fminf((b.top - l) * b.per_unit, (float)(b.n - 1));
}

// the bin at which the count (or mass) exceeds target: sh.found_bin / count / mass.  base_*: what lies before this thread's bins
template <bool BY_COUNT> __device__ void find_bin(const Bins& b, u64 base_mass, uint32_t base_count, u64 target, Shared& sh) {
  const int per = b.n / blockDim.x;
  for (int i = 0; i < per; ++i) {
    const int bin = threadIdx.x * per + i;
    const u64 m = b.mass[bin];
    const uint32_t c = BY_COUNT ? b.count[bin] : 0;
    const bool here = BY_COUNT ? base_count <= target && target < (u64)base_count + c : base_mass <= target && target < base_mass + m;
    if (here) sh.found_bin = bin, sh.found_count = base_count, sh.found_mass = base_mass;
    base_mass += m;
    base_count += c;
  }
  __syncthreads();
}

// the entry of bin sh.found_bin at which the count (or mass) exceeds target -> sh.found_*
template <int TYPE, bool LOCAL, bool BY_COUNT>
__device__ void find_entry(const Row<TYPE>& r, const Bins& b, const Scale& sc, u64 target, Shared& sh) {
  const int bin = (int)sh.found_bin;
  const u64 before_mass = sh.found_mass;
  const uint32_t before_count = sh.found_count;
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  const uint32_t room = b.n / 2;
  each_entry<TYPE, LOCAL>(r, [&](float l, int i) {
    if (bin_of(b, l) == bin) {
      const uint32_t at = atomicAdd(&sh.n, 1u);
      if (at < room) b.list[at] = place_of(l, i);
    }
  });
  __syncthreads();
  const uint32_t n = sh.n;
  __syncthreads();
  const u64 rest = target - (BY_COUNT ? before_count : before_mass);
  if (n <= 64) {
    if (threadIdx.x < n) sh.digit_mass[threadIdx.x] = mass_of(weight(sc, of_key((uint32_t)(b.list[threadIdx.x] >> 32))));
    if (threadIdx.x < 64) pick_of_64<BY_COUNT>(sh, b.list, sh.digit_mass, (int)n, rest, 0, 0);   // one wave's own writes
    __syncthreads();
  } else if (n <= room) {
    select<BY_COUNT>(sh, rest, [&](auto f) {
      for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const u64 place = b.list[i];
        f(place, mass_of(weight(sc, of_key((uint32_t)(place >> 32)))));
      }
    });
  } else {
    // more of the row in one bin than the list holds (equal logits, mostly): straight from the row, round by round
    select<BY_COUNT>(sh, rest, [&](auto f) {
      each_entry<TYPE, LOCAL>(r, [&](float l, int i) {
        if (bin_of(b, l) == bin) f(place_of(l, i), mass_of(weight(sc, l)));
      });
    });
  }
  if (threadIdx.x == 0) sh.found_mass += before_mass, sh.found_count += before_count;
  __syncthreads();
}

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
__device__ __forceinline__ void answer(const SampleArgs& a, int b, int id, double w, u64 S) {
  a.ids[b] = id;
  if (a.logp) a.logp[b] = (float)log(w * ONE / (double)S);
}
__device__ __forceinline__ void answer_none(const SampleArgs& a, int b) {
  a.ids[b] = -1;
  if (a.logp) a.logp[b] = -INFINITY;
}

// list[0 .. n) in ascending order; room: its size, a power of two.  All pairs up to 256 entries, a bitonic network beyond.
__device__ void sort_places(u64* list, int n, int room, Shared& sh) {
  const int tid = threadIdx.x, nt = blockDim.x;
  if (n <= 256) {
    const int e = tid & 255, parts = nt >> 8, part = tid >> 8;
    const u64 mine = e < n ? list[e] : 0;
    if (tid < 256) sh.digit_count[tid] = 0;
    __syncthreads();
    if (e < n) {
      uint32_t c = 0;
#pragma unroll 4
      for (int j = part; j < n; j += parts) c += list[j] < mine;
      if (parts > 1) atomicAdd(&sh.digit_count[e], c);
      else sh.digit_count[e] = c;
    }
    __syncthreads();
    if (tid < n) list[sh.digit_count[tid]] = mine;
    __syncthreads();
    return;
  }
  int size = 512;
  while (size < n) size *= 2;   // n <= room
  for (int i = n + tid; i < size; i += nt) list[i] = ~0ull;
  __syncthreads();
  for (int k = 2; k <= size; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      for (int i = tid; i < size / 2; i += nt) {
        const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
        const u64 x = list[lo], y = list[hi];
        if ((x > y) == ((lo & k) == 0)) list[lo] = y, list[hi] = x;
      }
      __syncthreads();
    }
}

// The answer from a sorted list of the row's first n entries of the walk, where nothing after them can be kept (they are all
// there is, or the first top_k).  cum: room for n masses; n <= 4 workgroups' threads.
__device__ void draw_from_sorted(const SampleArgs& a, int b, const u64* list, int n, u64* cum, const Scale& sc, const Settings& o, Shared& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, per = (n + blockDim.x - 1) / blockDim.x;
  u64 sum = 0, over = 0;
  for (int i = 0; i < per; ++i) {
    const int e = tid * per + i;
    if (e < n) {
      const double w = weight(sc, of_key((uint32_t)(list[e] >> 32)));
      const u64 m = mass_of(w);
      sum += m;
      if (w >= (double)o.min_p) over += m;
      cum[e] = sum;
    }
  }
  u64 base = wave_scan(sum, lane);
  if (lane == 63) sh.wave_u64[wv] = base;
  base -= sum;
  __syncthreads();
  u64 S = 0;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) {
    if (i < wv) base += sh.wave_u64[i];
    S += sh.wave_u64[i];
  }
  auto at_mass = [&](u64 t, auto f) {   // f(entry, mass up to and with it) for the entry at which the mass exceeds t
    u64 before = base;
    for (int i = 0; i < per; ++i) {
      const int e = tid * per + i;
      if (e < n) {
        const u64 upto = base + cum[e];
        if (before <= t && t < upto) f(e, upto);
        before = upto;
      }
    }
  };
  if (o.top_p < 1.0f) {
    at_mass(nucleus_target(o.top_p, S), [&](int, u64 upto) { sh.found_mass = upto; });
    __syncthreads();
    S = sh.found_mass;
  }
  if (o.min_p > 0.0f) {
    over = block_sum(over, sh);
    if (over < S) S = over;
  }
  if (S < ONE_MASS) S = ONE_MASS;   // the largest entry stays whatever is asked
  at_mass(draw_target(o.u, S), [&](int e, u64) { answer(a, b, (int)(uint32_t)list[e], weight(sc, of_key((uint32_t)(list[e] >> 32))), S); });
}

// The entries that can be among the k largest: every thread has its largest entry, and the k-th largest of those is no larger
// than the k-th largest of all.  256 bins over the threads' largest find it; entries of its bin and of those above it go to the
// list, unsorted.  -> how many (more than `room`: the list is not complete, or fewer than k threads have an entry)
template <int TYPE, bool LOCAL>
__device__ uint32_t gather_top(const Row<TYPE>& r, int k, float top, float own_max, u64* list, uint32_t room, int index0, Shared& sh) {
  const int tid = threadIdx.x, lane = tid & 63;
  float lowest = own_max > -INFINITY ? -own_max : -INFINITY, unused = 0.0f;
  block_max2(lowest, unused, sh);
  const float per_unit = 255.0f / fmaxf(top + lowest, 1e-30f);
  auto bin = [&](float l) { return l == top ? 0 : (int)fminf((top - l) * per_unit, 255.0f); };
  for (int i = tid; i < 256; i += blockDim.x) sh.digit_count[i] = 0;
  if (tid == 0) sh.n = 0, sh.found_bin = 256;
  __syncthreads();
  if (own_max > -INFINITY) atomicAdd(&sh.digit_count[bin(own_max)], 1u);
  __syncthreads();
  if (tid < 64) {
    uint32_t c[4], before = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = sh.digit_count[4 * lane + i], before += c[i];
    before = wave_scan(before, lane) - before;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (before < (uint32_t)k && (uint32_t)k <= before + c[i]) sh.found_bin = 4 * lane + i;
      before += c[i];
    }
  }
  __syncthreads();
  const int cut = (int)sh.found_bin;
  if (cut >= 256) return room + 1;
  each_entry<TYPE, LOCAL>(r, [&](float l, int i) {
    if (bin(l) <= cut) {
      const uint32_t at = atomicAdd(&sh.n, 1u);
      if (at < room) list[at] = place_of(l, index0 + i);
    }
  });
  __syncthreads();
  const uint32_t n = sh.n;
  __syncthreads();
  return n;
}

// Any settings: masses (and counts, where a rank is asked for) of the bins in one pass over the row, then each question goes to
// one bin and to one entry of it.
template <int TYPE, bool LOCAL>
__device__ void draw_by_bins(const SampleArgs& a, int b, const Row<TYPE>& r, Bins& bins, const Scale& sc, const Settings& o, Shared& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, per = bins.n / blockDim.x;
  const bool ranked = o.top_k > 0 && o.top_k < r.n;
  for (int i = tid; i < bins.n; i += blockDim.x) {
    bins.mass[i] = 0;
    if (ranked) bins.count[i] = 0;
  }
  __syncthreads();
  u64 over = 0;
  const double q = o.min_p;
  each_entry<TYPE, LOCAL>(r, [&](float l, int) {
    const double w = weight(sc, l);
    const u64 m = mass_of(w);
    const int bin = bin_of(bins, l);
    if (m) atomicAdd(&bins.mass[bin], m);
    if (ranked) atomicAdd(&bins.count[bin], 1u);
    if (w >= q) over += m;
  });
  __syncthreads();
  u64 base_mass = 0;
  uint32_t base_count = 0;
  for (int i = 0; i < per; ++i) {
    base_mass += bins.mass[tid * per + i];
    if (ranked) base_count += bins.count[tid * per + i];
  }
  const u64 own_mass = base_mass;
  const uint32_t own_count = base_count;
  base_mass = wave_scan(base_mass, lane);
  base_count = wave_scan(base_count, lane);
  if (lane == 63) sh.wave_u64[wv] = base_mass, sh.wave_u32[wv] = base_count;
  __syncthreads();
  base_mass -= own_mass;
  base_count -= own_count;
  u64 S = 0;
  uint32_t entries = 0;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) {
    if (i < wv) base_mass += sh.wave_u64[i], base_count += sh.wave_u32[i];
    S += sh.wave_u64[i];
    entries += sh.wave_u32[i];
  }
  __syncthreads();
  if (ranked && (uint32_t)o.top_k < entries) {
    find_bin<true>(bins, base_mass, base_count, o.top_k - 1, sh);
    find_entry<TYPE, LOCAL, true>(r, bins, sc, o.top_k - 1, sh);
    S = sh.found_mass + mass_of(weight(sc, of_key((uint32_t)(sh.found_place >> 32))));
    __syncthreads();
  }
  if (o.top_p < 1.0f) {
    const u64 t = nucleus_target(o.top_p, S);
    find_bin<false>(bins, base_mass, 0, t, sh);
    find_entry<TYPE, LOCAL, false>(r, bins, sc, t, sh);
    S = sh.found_mass + mass_of(weight(sc, of_key((uint32_t)(sh.found_place >> 32))));
    __syncthreads();
  }
  if (o.min_p > 0.0f) {
    over = block_sum(over, sh);
    if (over < S) S = over;
    __syncthreads();
  }
  if (S < ONE_MASS) S = ONE_MASS;   // the largest entry stays whatever is asked
  const u64 t = draw_target(o.u, S);
  find_bin<false>(bins, base_mass, 0, t, sh);
  find_entry<TYPE, LOCAL, false>(r, bins, sc, t, sh);
  if (tid == 0) answer(a, b, (int)(uint32_t)sh.found_place, weight(sc, of_key((uint32_t)(sh.found_place >> 32))), S);
}

// One workgroup a row, the row in shared memory (LOCAL) or read again for each pass.
template <int TYPE, bool LOCAL> __global__ __launch_bounds__(1024) void sample_row_kernel(SampleArgs a, int nbin) {
  typedef typename LOf<TYPE>::t T;
  extern __shared__ __align__(16) char dyn[];
  __shared__ Shared sh;
  const int b = blockIdx.x, tid = threadIdx.x;
  if (a.n_dev && b >= *a.n_dev) return;
  const int s = a.idx ? a.idx[b] : b;
  Row<TYPE> r((const T*)a.logits + (size_t)b * a.ld, a.V);
  Bins bins;
  bins.n = nbin;
  bins.mass = (u64*)dyn;
  bins.list = bins.mass + nbin;
  bins.count = (uint32_t*)bins.list;
  f32x4* local = (f32x4*)(bins.list + nbin / 2);
  float top = -INFINITY, low = -INFINITY;   // largest logit, largest negated finite one
  constexpr int EPC = Row<TYPE>::EPC;
#pragma unroll 4
  for (int c = tid; c < r.chunks; c += blockDim.x) {
    const Chunk<TYPE> k = r.global(c);
    if constexpr (LOCAL) local[c] = *(const f32x4*)k.v;
#pragma unroll
    for (int j = 0; j < EPC; ++j) {
      const float l = logit<TYPE>(k.v[j]);
      top = fmaxf(top, l);
      low = fmaxf(low, l > -INFINITY ? -l : -INFINITY);
    }
  }
  r.local = local;
  const float own_max = top;
  block_max2(top, low, sh);   // its barriers make the copy visible
  if (top == -INFINITY) {
    if (tid == 0) answer_none(a, b);
    return;
  }
  const Settings o = settings_of(a, s);
  if (!(o.temp > 0.0f) || o.top_k == 1) {   // the first of the largest
    if (tid == 0) sh.n = 0xffffffffu;
    __syncthreads();
    each_entry<TYPE, LOCAL>(r, [&](float l, int i) {
      if (l == top) atomicMin(&sh.n, (uint32_t)i);
    });
    __syncthreads();
    if (tid == 0) answer(a, b, (int)sh.n, 1.0, ONE_MASS);
    return;
  }
  const float temp = fminf(o.temp, 3.4e38f);
  const Scale sc = {top, 1.4426950408889634 / (double)temp};
  // few entries, or few that can be kept: sort them
  const int room = nbin / 2;
  if (a.V <= room || (o.top_k > 0 && o.top_k <= (int)blockDim.x / 2)) {
    uint32_t n;
    if (a.V <= room) {
      if (tid == 0) sh.n = 0;
      __syncthreads();
      each_entry<TYPE, LOCAL>(r, [&](float l, int i) { bins.list[atomicAdd(&sh.n, 1u)] = place_of(l, i); });
      __syncthreads();
      n = sh.n;
      __syncthreads();
    } else {
      n = gather_top<TYPE, LOCAL>(r, o.top_k, top, own_max, bins.list, room, 0, sh);
    }
    if (n <= (uint32_t)room) {
      sort_places(bins.list, (int)n, room, sh);
      draw_from_sorted(a, b, bins.list, o.top_k > 0 ? min((int)n, o.top_k) : (int)n, bins.mass, sc, o, sh);
      return;
    }
  }
  // bins down to 32 temperatures under the top (e^-32 < 2^-45: no mass beyond), or to the lowest logit if that is nearer
  bins.top = top;
  bins.per_unit = (float)nbin / fmaxf(fminf(32.0f * temp, top + low), 1e-30f);
  draw_by_bins<TYPE, LOCAL>(a, b, r, bins, sc, o, sh);
}

template <int TYPE, bool LOCAL> int launch_rows(const SampleArgs& a, int nbin, int threads, size_t lds, hipStream_t st) {
  ST_ENSURE_LDS((sample_row_kernel<TYPE, LOCAL>), 160 * 1024 - (int)sizeof(Shared));
  hipLaunchKernelGGL((sample_row_kernel<TYPE, LOCAL>), dim3(a.B), dim3(threads), lds, st, a, nbin);
  ST_LAUNCH_CHECK();
  return ST_OK;
}
template <int TYPE> int launch_type(const SampleArgs& a, hipStream_t st) {
  const size_t row = ((size_t)a.V * sizeof(typename LOf<TYPE>::t) + 31) / 16 * 16;
  const int nbin = a.V <= 1024 ? 2048 : a.V <= 16384 ? 1024 : a.V <= 65536 ? 2048 : 4096;
  const int threads = a.V <= 2048 ? 256 : a.B >= 1024 && a.V <= 16384 ? 512 : 1024;
  const size_t lds = (size_t)nbin * 12;
  if (lds + row <= 128 * 1024) return launch_rows<TYPE, true>(a, nbin, threads, lds + row, st);
  return launch_rows<TYPE, false>(a, nbin, threads, lds, st);
}

}  // namespace

size_t sample_workspace(int, int) { return 0; }

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
