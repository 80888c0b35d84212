// Products with 4-bit weights and group scales: y[m, n] = sum_k x[m, k] * s[n, k / g] * (c[n, k] - z[n, k / g]) + b[n].
//
// A weight is read as a code c in 0..15; c - z is a whole number in -15..15, which f16 holds exactly, so the matrix cores
// multiply f16 images of x with f16 whole numbers (v_mfma_f32_16x16x32_f16, sums in f32) and the scale is applied in f32 once a
// group: no weight is rounded.  x in f16 goes in as it is.  x in bf16 or f32 is first multiplied, row by row, with a power of
// two that brings the row's largest value to [2^14, 2^15).  A bf16 value then is an f16 value (8 significant bits of 11); what is
// below 2^-31 of the largest loses bits as an f16 subnormal, rounded to the nearest: an error of 2^-39 of the row's largest at
// most.  An f32 value is split into hi + lo and costs two products: hi is cut to 11 bits, what is left (below 2^-10 of the value's
// power of two) is rounded to the nearest of 11 bits: an error of 2^-22 of the value or, in subnormals, 2^-39 of the row's largest.
#include "st_common.h"

namespace {

constexpr int KB = 128;   // columns k of a block: 64 lanes x 16 bytes hold 16 rows n x 128 codes

struct Q4Layout {
  int sb, kb, gpb;         // blocks of 64 n, of 128 k; groups a block of k
  size_t scales, zeros, total;   // byte offsets
};

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

Q4Layout q4_layout(int N, int K, int group, int has_zeros) {
  Q4Layout y;
  y.sb = (N + 63) / 64;
  y.kb = (K + KB - 1) / KB;
  y.gpb = KB / group;
  const size_t blocks = (size_t)y.sb * y.kb;
  y.scales = blocks * 4096;
  y.zeros = y.scales + up256(blocks * 64 * y.gpb * 2);
  y.total = y.zeros + (has_zeros ? up256(blocks * 64 * y.gpb) : 0);
  return y;
}

int check_q4_shape(int N, int K, int group) {
  ST_CHECK_ARG(N > 0 && K > 0, "N=%d K=%d must be positive", N, K);
  ST_CHECK_ARG(N <= (1 << 24) && K <= (1 << 24), "N=%d K=%d: at most 2^24", N, K);
  ST_CHECK_ARG(group == 32 || group == 64 || group == 128, "group=%d unsupported (32, 64, 128)", group);
  return ST_OK;
}

// ---- image ---------------------------------------------------------------------------------------------------------------
// Block (sb, kb) holds 64 n x 128 k in four tiles of 16 n, 1 KB each: lane l's 16 bytes of tile t are the codes of row
// n = 64 sb + 16 t + (l & 15); its word j holds k = 128 kb + 32 j + 8 (l >> 4) + 0..7, the operand of one 16x16x32 product.  In the
// word, k's pair p (2p, 2p + 1) lies in the nibbles p and p + 4: one and-or makes a pair of f16 out of it.  Scales (f16) and zero
// codes (bytes) lie block by block, [16 l][4 t][groups of the block]: a lane reads those of its four rows at once.  Rows from N on
// and groups from K on have scale 0.
__global__ __launch_bounds__(256) void q4_pack_kernel(const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scales,
                                                      const uint8_t* __restrict__ zeros, int N, int K, int group, int kb_n, size_t tiles,
                                                      uint32_t* __restrict__ out, uint16_t* __restrict__ out_s, uint8_t* __restrict__ out_z) {
  const int row_bytes = (K + 1) / 2, groups = (K + group - 1) / group, gpb = KB / group;
  const int j = threadIdx.x & 3, lane = threadIdx.x >> 2;   // a workgroup a tile at a time, a thread a word
  for (size_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int t = (int)(tile & 3);
    const size_t b = tile >> 2;
    const int kb = (int)(b % kb_n), n = (int)(b / kb_n) * 64 + 16 * t + (lane & 15);
    const int k0 = kb * KB + 32 * j + 8 * (lane >> 4);
    uint32_t w = 0;
    if (n < N)
      for (int i = 0; i < 8; ++i) {
        const int k = k0 + i;
        if (k < K) {
          const uint32_t c = (codes[(size_t)n * row_bytes + (k >> 1)] >> (4 * (k & 1))) & 15u;
          w |= c << (4 * ((i >> 1) + 4 * (i & 1)));
        }
      }
    out[tile * 256 + threadIdx.x] = w;
    if (threadIdx.x < 16 * gpb) {
      const int l = threadIdx.x / gpb, i = threadIdx.x % gpb, row = (int)(b / kb_n) * 64 + 16 * t + l, g = kb * gpb + i;
      const size_t at = ((b * 16 + l) * 4 + t) * gpb + i;
      const bool in = row < N && g < groups;
      out_s[at] = in ? scales[(size_t)row * groups + g] : (uint16_t)0;
      if (out_z) out_z[at] = in ? (uint8_t)(zeros[(size_t)row * groups + g] & 15) : (uint8_t)0;
    }
  }
}

// ---- codes of an f32 matrix ------------------------------------------------------------------------------------------------
// One wave a (row, group).  Without zero codes: s = max |w| / 7 and z = 8; with them the range [min(w, 0), max(w, 0)] is cut into
// 15 steps and z is 0's place in it.  s is rounded to f16 first, the codes go by the rounded one.  A group with a NaN or an infinity
// has s NaN, one whose s is beyond f16 has s infinite, with the codes of 0: neither is taken for ordinary weights.
__global__ __launch_bounds__(256) void q4_quantize_kernel(const float* __restrict__ W, int N, int K, int group, uint8_t* __restrict__ codes,
                                                          _Float16* __restrict__ scales, uint8_t* __restrict__ zeros) {
  const int groups = (K + group - 1) / group, lane = threadIdx.x & 63;
  for (size_t wv = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6); wv < (size_t)N * groups; wv += (size_t)gridDim.x * 4) {
    const int n = (int)(wv / groups), g = (int)(wv % groups);
    const int k = g * group + 2 * lane;                 // lanes 0 .. group / 2 - 1 have two columns each
    const bool in0 = 2 * lane < group && k < K, in1 = 2 * lane < group && k + 1 < K;
    const float a = in0 ? W[(size_t)n * K + k] : 0.0f, b = in1 ? W[(size_t)n * K + k + 1] : 0.0f;
    const float hi = wave_max(fmaxf(fmaxf(a, b), 0.0f)), lo = -wave_max(fmaxf(fmaxf(-a, -b), 0.0f));
    const bool finite = !__any(!(fabsf(a) < INFINITY && fabsf(b) < INFINITY));
    const float step = !finite ? NAN : zeros ? (hi - lo) / 15.0f : fmaxf(hi, -lo) / 7.0f;
    const _Float16 s16 = (_Float16)step;
    const float s = (float)s16;
    const int z = zeros ? (s > 0.0f ? min(15, max(0, (int)rintf(-lo / s))) : 0) : 8;
    const int c0 = s > 0.0f ? min(15, max(0, (int)fminf(fmaxf(rintf(a / s), -16.0f), 16.0f) + z)) : z;
    const int c1 = s > 0.0f ? min(15, max(0, (int)fminf(fmaxf(rintf(b / s), -16.0f), 16.0f) + z)) : z;
    if (in0) codes[(size_t)n * ((K + 1) / 2) + (k >> 1)] = (uint8_t)(c0 | (in1 ? c1 << 4 : 0));
    if (lane == 0) {
      scales[wv] = s16;
      if (zeros) zeros[wv] = (uint8_t)z;
    }
  }
}

// ---- product ---------------------------------------------------------------------------------------------------------------
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 8 codes -> 8 f16 values c - z.  0x6400 | c is the f16 1024 + c, and 0x5400 | c << 4 is 64 + c; both corrections are exact.  The
// masks lie in registers (the empty asm keeps hipcc from making literals of them): an and-or then is one instruction, and 8 codes
// take 9 instead of 13, which is what a product with few rows has to do per weight.
struct Open {
  uint32_t low, high, b_low, b_high;
  __device__ __forceinline__ Open() : low(0x000f000fu), high(0x00f000f0u), b_low(0x64006400u), b_high(0x54005400u) {
    asm("" : "+v"(low), "+v"(high), "+s"(b_low), "+s"(b_high));
  }
  __device__ __forceinline__ h8 operator()(uint32_t w, h2 z_low, h2 z_high) const {
    const uint32_t v = w >> 8;
    const h2 a = __builtin_bit_cast(h2, (w & low) | b_low) + z_low, b = __builtin_bit_cast(h2, (w & high) | b_high) + z_high;
    const h2 c = __builtin_bit_cast(h2, (v & low) | b_low) + z_low, d = __builtin_bit_cast(h2, (v & high) | b_high) + z_high;
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
};

template <int TYPE> struct XOf;
template <> struct XOf<ST_TYPE_F32> { typedef float t; };
template <> struct XOf<ST_TYPE_BF16> { typedef uint16_t t; };
template <> struct XOf<ST_TYPE_F16> { typedef _Float16 t; };

// a barrier for shared memory alone: loads from global memory stay under way across it (__syncthreads waits for them)
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

struct Q4Args {
  const void* x;
  long ldx;
  const void* x8;   // where 8 values at a time are read from, at columns up to k8: x and K - 8; with K < 8 any memory (the image)
  long ldx8;
  int k8;
  int M, N, K, nb, kb;
  const u32x4* codes;
  const void* scales;
  const void* zeros;
  const float* bias;
  void* y;
  long ldy;
};

__device__ __forceinline__ uint16_t bf16_of(float v) {   // nearest, ties to even; NaN stays NaN
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}
template <int TYPE> __device__ __forceinline__ void store_y(const Q4Args& a, int row, int n, float v) {
  typedef typename XOf<TYPE>::t T;
  T* y = (T*)a.y + (size_t)row * a.ldy + n;
  if constexpr (TYPE == ST_TYPE_BF16) *y = bf16_of(v);
  else *y = (T)v;
}

// ---- x ---------------------------------------------------------------------------------------------------------------------
// 8 values of a row from column k on, as they lie in memory (any alignment); columns from K on are 0
template <int TYPE> struct X8 {
  uint32_t w[TYPE == ST_TYPE_F32 ? 8 : 4];
  // no branch stands around a load, so that it can stay under way: where fewer than 8 columns are left the row's last 8 are read,
  // and whoever uses them comes back for the right ones (tail)
  __device__ __forceinline__ void load(const Q4Args& a, const typename XOf<TYPE>::t* p8, int k) { __builtin_memcpy(w, p8 + min(k, a.k8), sizeof(w)); }
  __device__ __forceinline__ void tail(const Q4Args& a, const typename XOf<TYPE>::t* p, int k) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(w) / 4); ++i) {
      if constexpr (TYPE == ST_TYPE_F32) {
        w[i] = k + i < a.K ? __float_as_uint(p[k + i]) : 0;
      } else {
        const uint32_t lo = k + 2 * i < a.K ? ((const uint16_t*)p)[k + 2 * i] : 0;
        const uint32_t hi = k + 2 * i + 1 < a.K ? ((const uint16_t*)p)[k + 2 * i + 1] : 0;
        w[i] = lo | hi << 16;
      }
    }
  }
  __device__ __forceinline__ float value(int i) const {   // not for f16
    if constexpr (TYPE == ST_TYPE_F32) return __uint_as_float(w[i]);
    else return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
  }
  __device__ __forceinline__ float largest(float m) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(value(i)));
    return m;
  }
  // the values times 2^14 over the row's power of two as f16, and for f32 what that leaves
  __device__ __forceinline__ void split(float shift, h8& hi, h8& lo) const {
    if constexpr (TYPE == ST_TYPE_F16) {
      hi = __builtin_bit_cast(h8, *(const u32x4*)w);
    } else {
      uint32_t h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = value(2 * i) * shift, b = value(2 * i + 1) * shift;
        // f32: towards 0, what that leaves is kept in lo (to the nearest here takes 7 x 4751 x 2119 from 8.5 to 9.4 us)
        const h2 q = TYPE == ST_TYPE_F32 ? __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(a, b)) : h2{(_Float16)a, (_Float16)b};
        h[i] = __builtin_bit_cast(uint32_t, q);
        if constexpr (TYPE == ST_TYPE_F32) {
          lo[2 * i] = (_Float16)fmaxf(a - (float)q[0], -65504.0f);        // an infinity: inf - inf is not wanted
          lo[2 * i + 1] = (_Float16)fmaxf(b - (float)q[1], -65504.0f);
        }
      }
      hi = __builtin_bit_cast(h8, *(const u32x4*)h);
    }
  }
};
// The exponent field of a row's largest value so far, 15 at least: 2^(141 - e) brings values of that size to [2^14, 2^15)
__device__ __forceinline__ int exponent_of(float big) { return (int)((__float_as_uint(big) >> 23) & 255); }
__device__ __forceinline__ float shift_of(int e) { return __uint_as_float((uint32_t)(268 - e) << 23); }
__device__ __forceinline__ float unshift_of(int e) { return __uint_as_float((uint32_t)(e - 14) << 23); }
__device__ __forceinline__ float shrink_of(int from, int to) { return to - from > 126 ? 0.0f : __uint_as_float((uint32_t)(127 - (to - from)) << 23); }

// ---- weights ---------------------------------------------------------------------------------------------------------------
// what one lane holds of NT tiles of a block: codes, and the block's scales and zero codes of its rows
template <int BYTES> __device__ __forceinline__ void load_bytes(uint32_t* w, const void* p) {
  if constexpr (BYTES == 1) w[0] = *(const uint8_t*)p;
  else if constexpr (BYTES == 2) w[0] = *(const uint16_t*)p;
  else __builtin_memcpy(w, __builtin_assume_aligned(p, BYTES < 16 ? BYTES : 16), BYTES);
}
template <int GPB, int NT> struct W8 {
  u32x4 codes[NT];
  uint32_t s[(NT * GPB + 1) / 2], z[(NT * GPB + 3) / 4];
  __device__ __forceinline__ void load(const Q4Args& a, int nb, int kb, int lane) {   // nb: a multiple of NT
    const size_t blk = (size_t)(nb >> 2) * a.kb + kb, at = (blk * 64 + (lane & 15) * 4 + (nb & 3)) * GPB;
    const u32x4* c = a.codes + (blk * 4 + (nb & 3)) * 64 + lane;
#pragma unroll
    for (int t = 0; t < NT; ++t) codes[t] = c[64 * t];
    load_bytes<NT * GPB * 2>(s, (const char*)a.scales + at * 2);
    // (no branch here either: without zero codes the scales are read, and dropped)
    load_bytes<NT * GPB>(z, (const char*)(a.zeros ? a.zeros : a.scales) + at);
  }
  __device__ __forceinline__ void settle(const Q4Args& a) {   // before the first use
#pragma unroll
    for (int i = 0; i < (NT * GPB + 3) / 4; ++i) z[i] = a.zeros ? z[i] : 0x08080808u;
  }
  __device__ __forceinline__ float scale(int t, int g) const {
    const int i = t * GPB + g;
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(s[i >> 1] >> (16 * (i & 1))));
  }
  // the f16 pairs -1024 - z and -64 - z: 0xe400 | z and 0xd400 | z << 4
  __device__ __forceinline__ h2 zero_low(int t, int g) const {
    const int i = t * GPB + g;
    const uint32_t v = (z[i >> 2] >> (8 * (i & 3))) & 15u;
    return __builtin_bit_cast(h2, 0xe400e400u | v | v << 16);
  }
  __device__ __forceinline__ h2 zero_high(int t, int g) const {
    const int i = t * GPB + g;
    const uint32_t v = (z[i >> 2] >> (8 * (i & 3))) & 15u;
    return __builtin_bit_cast(h2, 0xd400d400u | v << 4 | v << 20);
  }
};

// One workgroup: 16 rows m x 16 NT columns n; its waves take the k blocks in turn and are joined through shared memory.  For few
// rows: what bounds it is reading the weights, once, with a block of every wave under way while the last one is multiplied.
template <int TYPE, int GPB, int NT, bool ONE>   // ONE: a block a wave
__global__ __launch_bounds__(512) void q4_rows_kernel(Q4Args a) {
  extern __shared__ float red[];   // [waves][NT][4][64]
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const int kq = 8 * (lane >> 4), quad = lane >> 4;
  const int nb0 = blockIdx.x * NT;
  // lanes of absent rows read the last one: nothing comes of it
  typedef typename XOf<TYPE>::t T;
  const size_t row = min((int)blockIdx.y * 16 + (lane & 15), a.M - 1);
  const T *xrow = (const T*)a.x + row * a.ldx, *xrow8 = (const T*)a.x8 + row * a.ldx8;
  struct Stage {
    W8<GPB, NT> w;
    X8<TYPE> x[4];
  };
  auto load = [&](Stage& s, int b) __attribute__((always_inline)) {
    s.w.load(a, nb0, b, lane);
#pragma unroll
    for (int j = 0; j < 4; ++j) s.x[j].load(a, xrow8, b * KB + 32 * j + kq);
  };
  const Open open;
  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = f32x4{0, 0, 0, 0};
  int e = 15;
  auto multiply = [&](Stage& cur, int b) __attribute__((always_inline)) {
    if ((b + 1) * KB > a.K) {
#pragma unroll
      for (int j = 0; j < 4; ++j) cur.x[j].tail(a, xrow, b * KB + 32 * j + kq);
    }
    cur.w.settle(a);
    float shift = 1.0f;
    if constexpr (TYPE != ST_TYPE_F16) {
      float big = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) big = cur.x[j].largest(big);
      big = fmaxf(big, __shfl_xor(big, 16, 64));
      big = fmaxf(big, __shfl_xor(big, 32, 64));
      const int e1 = max(e, min(254, exponent_of(big)));
      if (b != wv && __any(e1 != e)) {   // rows m of the product are 4 quad + i: their sums so far shrink to the new power of two
        const float f = shrink_of(e, e1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float fi = __shfl(f, 4 * quad + i, 64);
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[t][i] *= fi;
        }
      }
      e = e1;
      shift = shift_of(e);
    }
    f32x4 part[NT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h8 xh, xl;
      cur.x[j].split(shift, xh, xl);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int g = j * GPB / 4;
        const h8 w = open(cur.w.codes[t][j], cur.w.zero_low(t, g), cur.w.zero_high(t, g));
        const bool first = j % (4 / GPB) == 0, last = (j + 1) % (4 / GPB) == 0;
        part[t] = mfma16x32h(xh, w, first ? f32x4{0, 0, 0, 0} : part[t]);
        if constexpr (TYPE == ST_TYPE_F32) part[t] = mfma16x32h(xl, w, part[t]);
        if (last) acc[t] += part[t] * cur.w.scale(t, g);
      }
    }
  };
  Stage cur;
  load(cur, wv);
  if constexpr (ONE) {
    multiply(cur, wv);
  } else {
#pragma unroll 1
    for (int b = wv;; b += nw) {
      const bool more = b + nw < a.kb;
      Stage next;
      if (more) load(next, b + nw);
      multiply(cur, b);
      if (!more) break;
      cur = next;
    }
  }
  const float unshift = TYPE == ST_TYPE_F16 ? 1.0f : unshift_of(e);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float f = TYPE == ST_TYPE_F16 ? 1.0f : __shfl(unshift, 4 * quad + i, 64);
#pragma unroll
    for (int t = 0; t < NT; ++t) red[((wv * NT + t) * 4 + i) * 64 + lane] = acc[t][i] * f;
  }
  __syncthreads();
  for (int o = threadIdx.x; o < NT * 256; o += blockDim.x) {
    const int r = o / (16 * NT), col = o % (16 * NT), row = blockIdx.y * 16 + r, n = nb0 * 16 + col;
    if (row >= a.M || n >= a.N) continue;
    const int src = ((col >> 4) * 4 + (r & 3)) * 64 + 16 * (r >> 2) + (col & 15);
    float s = a.bias ? a.bias[n] : 0.0f;
    for (int q = 0; q < nw; ++q) s += red[q * NT * 256 + src];
    store_y<TYPE>(a, row, n, s);
  }
}

// One workgroup: 16 MT WM rows m x 16 NT WN columns n, WM x WN waves of MT x NT tiles each, for more than 16 rows.  Every block of
// 128 k of x is brought to f16 once a workgroup, a thread a row's quarter, into the operand order of the matrix instruction
// (a wave reads 1 KB in a row: no bank conflicts), in two buffers, so that one barrier a block is enough; the weights go from global
// memory to registers, a block ahead.
template <int TYPE, int GPB, int MT, int NT, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void q4_tile_kernel(Q4Args a, int tiles_m, int tiles_n) {
  constexpr int ROWS = 16 * MT * WM, PARTS = TYPE == ST_TYPE_F32 ? 2 : 1, WAVES = WM * WN, UNITS = ROWS / 16 / WAVES;
  static_assert(UNITS * WAVES * 16 == ROWS, "every wave stages UNITS times 16 rows");
  extern __shared__ __align__(16) char dyn[];
  h8* const xs = (h8*)dyn;                                            // [2][PARTS][ROWS / 16][4][64]
  float* const shrink = (float*)(xs + 2 * PARTS * ROWS * 16);         // [2][ROWS]
  int* const shrunk = (int*)(shrink + 2 * ROWS);                      // [2]: the block that the buffer's factors belong to
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, quad = lane >> 4;
  // tiles of the same columns on the same XCD (workgroups go round the eight of them): its L2 has the weights once
  const int xcd = blockIdx.x & 7, idx = blockIdx.x >> 3, tile_n = idx / tiles_m * 8 + xcd, tile_m = idx % tiles_m;
  if (tile_n >= tiles_n) return;
  const int m0 = tile_m * ROWS, wm = wv / WN, wn = wv % WN, nb0 = (tile_n * WN + wn) * NT;
  const int nbl = min(nb0, (a.nb - 1) & ~(NT - 1));                  // waves behind the last column read the last ones again
  // staging: this thread's rows 16 (wv + WAVES u) + (lane & 15) and their columns 8 quad + 32 j
  typedef typename XOf<TYPE>::t T;
  const int kq = 8 * quad;
  int e[UNITS];
  X8<TYPE> raw[UNITS][4];
  size_t row[UNITS];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) row[u] = min(m0 + 16 * (wv + WAVES * u) + (lane & 15), a.M - 1), e[u] = 15;
  auto load_x = [&](int b) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) raw[u][j].load(a, (const T*)a.x8 + row[u] * a.ldx8, b * KB + 32 * j + kq);
  };
  auto stage = [&](int b) __attribute__((always_inline)) {
    const int buf = b & 1;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int rb = wv + WAVES * u;
      if ((b + 1) * KB > a.K) {
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[u][j].tail(a, (const T*)a.x + row[u] * a.ldx, b * KB + 32 * j + kq);
      }
      float shift = 1.0f;
      if constexpr (TYPE != ST_TYPE_F16) {
        float big = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) big = raw[u][j].largest(big);
        big = fmaxf(big, __shfl_xor(big, 16, 64));
        big = fmaxf(big, __shfl_xor(big, 32, 64));
        const int e1 = max(e[u], min(254, exponent_of(big)));
        if (quad == 0) shrink[buf * ROWS + 16 * rb + (lane & 15)] = shrink_of(e[u], e1);
        if (__any(e1 != e[u]) && lane == 0) shrunk[buf] = b;
        e[u] = e1;
        shift = shift_of(e1);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        h8 hi, lo;
        raw[u][j].split(shift, hi, lo);
        xs[((buf * PARTS + 0) * (ROWS / 16) + rb) * 256 + j * 64 + lane] = hi;
        if constexpr (PARTS == 2) xs[((buf * PARTS + 1) * (ROWS / 16) + rb) * 256 + j * 64 + lane] = lo;
      }
    }
  };
  const Open open;
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0, 0, 0, 0};
  if (tid < 2) shrunk[tid] = 0;   // block 0 shrinks sums that are still 0
  auto multiply = [&](W8<GPB, NT>& cur, int b) __attribute__((always_inline)) {
    const int buf = b & 1;
    cur.settle(a);
    if (TYPE != ST_TYPE_F16 && b > 0 && shrunk[buf] == b) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const f32x4 f = *(const f32x4*)&shrink[buf * ROWS + (wm * MT + i) * 16 + 4 * quad];
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] *= f;
      }
    }
    f32x4 part[MT][NT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      constexpr int JG = 4 / GPB;
      const int g = j / JG;
      const bool first = j % JG == 0, last = (j + 1) % JG == 0;
      h8 xh[MT], xl[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        xh[i] = xs[((buf * PARTS + 0) * (ROWS / 16) + wm * MT + i) * 256 + j * 64 + lane];
        if constexpr (PARTS == 2) xl[i] = xs[((buf * PARTS + 1) * (ROWS / 16) + wm * MT + i) * 256 + j * 64 + lane];
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const h8 w = open(cur.codes[t][j], cur.zero_low(t, g), cur.zero_high(t, g));
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          part[i][t] = mfma16x32h(xh[i], w, first ? f32x4{0, 0, 0, 0} : part[i][t]);
          if constexpr (PARTS == 2) part[i][t] = mfma16x32h(xl[i], w, part[i][t]);
        }
      }
      if (last) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float s = cur.scale(t, g);
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[i][t] += part[i][t] * s;
        }
      }
    }
  };
  W8<GPB, NT> even, odd;
  const int last_b = a.kb - 1;
  load_x(0);
  even.load(a, nbl, 0, lane);
  __syncthreads();
  stage(0);
#pragma unroll 1
  for (int b = 0;; b += 2) {
    lds_barrier();   // block b is staged, and nobody reads the other buffer any more
    load_x(min(b + 1, last_b));
    odd.load(a, nbl, min(b + 1, last_b), lane);
    __builtin_amdgcn_sched_barrier(0);   // they go out before the products
    multiply(even, b);
    if (b + 1 > last_b) break;
    stage(b + 1);
    lds_barrier();
    load_x(min(b + 2, last_b));
    even.load(a, nbl, min(b + 2, last_b), lane);
    __builtin_amdgcn_sched_barrier(0);
    multiply(odd, b + 1);
    if (b + 2 > last_b) break;
    stage(b + 2);
  }
  __syncthreads();
  if (TYPE != ST_TYPE_F16 && quad == 0) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) shrink[16 * (wv + WAVES * u) + (lane & 15)] = unshift_of(e[u]);
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = (nb0 + t) * 16 + (lane & 15);
    if (n >= a.N) continue;
    const float bias = a.bias ? a.bias[n] : 0.0f;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int r = (wm * MT + i) * 16 + 4 * quad;
      const f32x4 f = TYPE == ST_TYPE_F16 ? f32x4{1, 1, 1, 1} : *(const f32x4*)&shrink[r];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (m0 + r + c < a.M) store_y<TYPE>(a, m0 + r + c, n, acc[i][t][c] * f[c] + bias);
    }
  }
}

template <int TYPE, int GPB, int MT, int NT, int WM, int WN> int launch_tile(const Q4Args& a, hipStream_t st) {
  constexpr int ROWS = 16 * MT * WM, COLS = NT * WN, PARTS = TYPE == ST_TYPE_F32 ? 2 : 1;
  constexpr int lds = 2 * PARTS * ROWS * 256 + 2 * ROWS * 4 + 16;
  const int tiles_m = (a.M + ROWS - 1) / ROWS, tiles_n = (a.nb + COLS - 1) / COLS;
  const long grid = (long)(tiles_n + 7) / 8 * 8 * tiles_m;
  ST_CHECK_ARG(grid * 64 * WM * WN < (1L << 32), "M=%d N=%d: too large for one launch", a.M, a.N);
  ST_ENSURE_LDS((q4_tile_kernel<TYPE, GPB, MT, NT, WM, WN>), lds);
  hipLaunchKernelGGL((q4_tile_kernel<TYPE, GPB, MT, NT, WM, WN>), dim3((unsigned)grid), dim3(64 * WM * WN), lds, st, a, tiles_m, tiles_n);
  ST_LAUNCH_CHECK();
  return ST_OK;
}
template <int TYPE, int GPB, int NT> int launch_rows(const Q4Args& a, hipStream_t st) {
  const int nw = a.kb < 8 ? a.kb : 8;
  const dim3 grid((a.nb + NT - 1) / NT, (a.M + 15) / 16), block(64 * nw);
  const size_t lds = (size_t)nw * NT * 1024;
  if (a.kb <= nw) hipLaunchKernelGGL((q4_rows_kernel<TYPE, GPB, NT, true>), grid, block, lds, st, a);
  else hipLaunchKernelGGL((q4_rows_kernel<TYPE, GPB, NT, false>), grid, block, lds, st, a);
  ST_LAUNCH_CHECK();
  return ST_OK;
}
// Which kernel, measured on both sides (f16 / f32, us): the rows kernel reads and opens every weight once for each 16 rows and has
// a short way for each, the tile kernel once for each 64 or 128, behind a barrier a block of k.  16 x 16 x 128 blocks of the product:
// 65 536 (128 x 8192 x 2048) 19.8 / 32.8 by rows, 22.7 / 39.4 by tiles; 131 072 (256 x 4096 x 4096) 32 / 57, 37 / 69; 262 144
// (128 x 16384 x 4096) 63 / 113, 39 / 71.  The large tile, where a launch of it fills the chip: 256 x 32768 x 4096 91 / 214 against
// 109 / 276; with half as many workgroups (128 x 16384 x 4096) it takes 81 / 104 against 39 / 71.
template <int TYPE, int GPB> int q4_launch(const Q4Args& a, hipStream_t st) {
  const long mt = (a.M + 15) / 16;
  if (mt > 1 && mt * a.nb * a.kb >= 196608) {
    constexpr int NT = TYPE == ST_TYPE_F32 ? 2 : 4;
    if ((mt + 7) / 8 * ((a.nb + 4 * NT - 1) / (4 * NT)) >= 192) return launch_tile<TYPE, GPB, 4, NT, 2, 4>(a, st);
    return launch_tile<TYPE, GPB, 4, 2, 1, 4>(a, st);
  }
  // tiles of a wave: one while the launch has fewer than two waves a SIMD and more (4096 x 4096 on one row: 5.2 us, 6.1 with two,
  // 8.3 with four), four where x is brought to f16 for many (16384 x 4096: 17, 14, 12 us)
  const long waves = a.nb * (a.kb < 8 ? a.kb : 8) * mt;
  if (waves >= 8192) return launch_rows<TYPE, GPB, 4>(a, st);
  if (waves >= 4096) return launch_rows<TYPE, GPB, 2>(a, st);
  return launch_rows<TYPE, GPB, 1>(a, st);
}
template <int TYPE> int q4_launch_group(const Q4Args& a, int group, hipStream_t st) {
  return group == 32 ? q4_launch<TYPE, 4>(a, st) : group == 64 ? q4_launch<TYPE, 2>(a, st) : q4_launch<TYPE, 1>(a, st);
}

}  // namespace

extern "C" size_t st_q4_packed_bytes(int N, int K, int group, int has_zeros) {
  if (N <= 0 || K <= 0 || N > (1 << 24) || K > (1 << 24) || (group != 32 && group != 64 && group != 128)) return 0;
  return q4_layout(N, K, group, has_zeros).total;
}

// workgroups of 256 threads for so many pieces of a weight: a launch has fewer than 2^32 threads, beyond 2^23 a workgroup takes several
static unsigned weight_blocks(size_t pieces) { return (unsigned)(pieces < (1u << 23) ? pieces : 1u << 23); }

extern "C" int st_pack_weight_q4(const uint8_t* codes, const void* scales, const uint8_t* zeros, int N, int K, int group, void* out_packed,
                                 void* stream) {
  ST_TRY(check_q4_shape(N, K, group));
  ST_CHECK_ARG(codes && scales && out_packed, "NULL buffer");
  ST_CHECK_ARG(((size_t)out_packed & 15) == 0, "the packed image must lie on 16 bytes");
  const Q4Layout y = q4_layout(N, K, group, zeros != nullptr);
  const size_t tiles = (size_t)y.sb * y.kb * 4;
  char* out = (char*)out_packed;
  hipLaunchKernelGGL(q4_pack_kernel, dim3(weight_blocks(tiles)), dim3(256), 0, (hipStream_t)stream, codes, (const uint16_t*)scales,
                     zeros, N, K, group, y.kb, tiles, (uint32_t*)out, (uint16_t*)(out + y.scales), zeros ? (uint8_t*)(out + y.zeros) : nullptr);
  ST_LAUNCH_CHECK();
  return ST_OK;
}

extern "C" int st_quantize_weight_q4(const float* W, int N, int K, int group, uint8_t* codes, void* scales, uint8_t* zeros, void* stream) {
  ST_TRY(check_q4_shape(N, K, group));
  ST_CHECK_ARG(W && codes && scales, "NULL buffer");
  const size_t waves = (size_t)N * ((K + group - 1) / group);
  hipLaunchKernelGGL(q4_quantize_kernel, dim3(weight_blocks((waves + 3) / 4)), dim3(256), 0, (hipStream_t)stream, W, N, K, group, codes,
                     (_Float16*)scales, zeros);
  ST_LAUNCH_CHECK();
  return ST_OK;
}

extern "C" int st_gemm_q4(const void* x, int type, int64_t ldx, int M, const StQ4Weight* w, const float* bias, void* y, int64_t ldy,
                          void* stream) {
  ST_CHECK_ARG(w != nullptr, "weights struct is NULL");
  ST_TRY(check_q4_shape(w->N, w->K, w->group));
  ST_CHECK_ARG(type == ST_TYPE_F32 || type == ST_TYPE_BF16 || type == ST_TYPE_F16, "type=%d unknown", type);
  ST_CHECK_ARG(M >= 0 && M <= ST_Q4_MAX_ROWS, "M=%d (0 .. %d)", M, ST_Q4_MAX_ROWS);
  if (M == 0) return ST_OK;
  ST_CHECK_ARG(x && w->image && y, "NULL buffer");
  ST_CHECK_ARG(((size_t)w->image & 15) == 0, "the packed image must lie on 16 bytes");
  const size_t size = type == ST_TYPE_F32 ? 4 : 2;
  ST_CHECK_ARG(((size_t)x & (size - 1)) == 0 && ((size_t)y & (size - 1)) == 0, "x and y must lie on their type's size");
  ST_CHECK_ARG(ldx >= 0 && (M == 1 || ldy >= w->N), "ldx=%lld ldy=%lld: negative, or rows of y (%d values) overlap", (long long)ldx, (long long)ldy, w->N);
  const Q4Layout l = q4_layout(w->N, w->K, w->group, w->has_zeros);
  Q4Args a;
  a.x = x; a.ldx = M == 1 ? w->K : ldx; a.M = M; a.N = w->N; a.K = w->K; a.nb = (w->N + 15) / 16; a.kb = l.kb;
  a.codes = (const u32x4*)w->image;
  a.scales = (const char*)w->image + l.scales;
  a.zeros = w->has_zeros ? (const char*)w->image + l.zeros : nullptr;
  a.x8 = w->K >= 8 ? x : w->image; a.ldx8 = w->K >= 8 ? a.ldx : 0; a.k8 = w->K >= 8 ? w->K - 8 : 0;
  a.bias = bias; a.y = y; a.ldy = M == 1 ? w->N : ldy;
  hipStream_t st = (hipStream_t)stream;
  return type == ST_TYPE_F32 ? q4_launch_group<ST_TYPE_F32>(a, w->group, st)
         : type == ST_TYPE_BF16 ? q4_launch_group<ST_TYPE_BF16>(a, w->group, st) : q4_launch_group<ST_TYPE_F16>(a, w->group, st);
}
