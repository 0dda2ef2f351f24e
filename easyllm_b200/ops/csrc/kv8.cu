// A key/value cache held in 8 bits: written, read back, attended over.
//
// Rows k [R, G, dk], v [R, G, dv] of int8 (dk, dv: the head sizes rounded up to 16), and a scale for each block of `block` rows
// and head, [R / block, G], fp32.  A scale is a power of two s = 2^e, e >= -126, the least with max|x| <= 127 s (at most 2^121, where
// q is cut to 127: 128 2^121 is past the end of fp32 and bf16); x = q s, |q| <= 127.
// So x / s and q s_old / s are exact but for one rounding to an integer, and q s is exact in bf16 and in fp32: reading back loses
// nothing, and a block that rows join later is off by less than s (s / 2 + s / 4 + ..: a scale that grows at least doubles).
// A block that got a value that is not finite has the scale NaN and reads as NaN.
#include <algorithm>

#include "sm100.cuh"
#include "vec.cuh"

namespace ell {

constexpr int kK8Place = 51;      // error word: a sequence lies outside the cache or starts inside a block
constexpr int kK8Dim = 128, kK8MaxBlock = 128;

struct Kv8Cache {
  int8_t *k, *v;
  float *ks, *vs;
  long long rows;
  int G, d, dv, shift;            // block = 1 << shift
};
__host__ __device__ __forceinline__ int k8_row(int d) { return (d + 15) / 16 * 16; }

// Whether `n` rows from `base` on lie in the cache, from the start of a block.
__device__ __forceinline__ bool k8_inside(const Kv8Cache& c, int base, int n) {
  return base >= 0 && (base & ((1 << c.shift) - 1)) == 0 && (long long)base + n <= c.rows;
}
__device__ __forceinline__ float k8_scale_of(float amax) {       // amax finite, >= 0
  const int e = (int)((__float_as_uint(amax) + 0x1ffffu) >> 23) - 6;      // 127 = 2^6 (2 - 2^-6): carries above that mantissa
  return __uint_as_float((uint32_t)min(max(e, 1), 127 + 121) << 23);
}
__device__ __forceinline__ float k8_nan() { return __int_as_float(0x7fffffff); }

// ---- writing -----------------------------------------------------------------------------------
// A warp a block of a sequence, head, and keys or values.  Rows of the block that the step does not bring stay, requantised where the
// scale grows.
template <typename T>
__global__ void __launch_bounds__(256) kv8_append_kernel(const Kv8Cache c, const T* __restrict__ k, const T* __restrict__ v, const int* __restrict__ base_,
                                                         const int* __restrict__ len_, const int* __restrict__ cu, int n_seq, int n, int blocks,
                                                         int ldk, int ldv, int* __restrict__ err) {
  chain_enter(k, v, base_, len_, cu, err);
  const long long item = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, g = (int)(item % c.G);
  const long long rest = item / c.G;
  const int which = (int)(rest & 1), j = (int)((rest >> 1) % blocks);
  const long long s = (rest >> 1) / blocks;
  if (s >= n_seq) return;
  const int r0 = cu[s], count = min(cu[s + 1], n) - r0;
  if (count <= 0 || r0 < 0) return;
  const int base = base_[r0], p0 = len_[r0] - 1;
  if (p0 < 0) return;                                             // a padding row
  const int b = (p0 >> c.shift) + j, first = max(p0, b << c.shift), last = min(p0 + count, (b + 1) << c.shift);
  if (first >= last) return;
  if (!k8_inside(c, base, p0 + count)) {
    if (lane == 0) atomicCAS(err, 0, kK8Place);
    return;
  }
  const int width = which ? c.dv : c.d, row = k8_row(width), ld = which ? ldv : ldk;
  const T* src = (which ? v : k) + (size_t)r0 * ld + (size_t)g * width;
  int8_t* dst = (which ? c.v : c.k) + ((size_t)base * c.G + g) * row;
  float* scale = (which ? c.vs : c.ks) + ((size_t)(base >> c.shift) + b) * c.G + g;
  float amax = 0.f;
  bool odd = false;
  for (int p = first; p < last; ++p)
    for (int x = lane; x < width; x += 32) {
      const float f = fabsf(to_f<T>(src[(size_t)(p - p0) * ld + x]));
      odd = odd || !(f <= 3.4028235e38f);
      amax = fmaxf(amax, f);
    }
  odd = __any_sync(0xffffffffu, odd);
  float now = odd ? k8_nan() : k8_scale_of(warp_max(amax));
  const int start = b << c.shift;
  if (first > start) {                                            // rows that were there
    const float old = *scale;
    const bool grows = !(old >= now);
    if (old != old || odd) now = k8_nan();
    else if (!grows) now = old;
    if (grows && now == now) {
      const float f = old / now;
      for (int p = start; p < first; ++p)
        for (int x = lane; x < row; x += 32) {
          int8_t* q = dst + (size_t)p * c.G * row + x;
          *q = (int8_t)__float2int_rn((float)*q * f);
        }
    }
  }
  const float inv = 1.f / now;                                    // a power of two
  for (int p = first; p < last; ++p)
    for (int x = lane; x < row; x += 32) {
      float f = 0.f;
      if (x < width && now == now) f = fminf(fmaxf(to_f<T>(src[(size_t)(p - p0) * ld + x]) * inv, -127.f), 127.f);
      dst[(size_t)p * c.G * row + x] = (int8_t)__float2int_rn(f);
    }
  __syncwarp();                                                   // everybody has read the old scale
  if (lane == 0) *scale = now;
}

// ---- reading back ------------------------------------------------------------------------------
// ko [n, max_len, G, d], vo [n, max_len, G, dv]: rows base[i] .. base[i] + len[i] - 1, then zeros.  Eight values a thread (V) or one.
template <typename T, int V>
__global__ void __launch_bounds__(256) kv8_read_kernel(const Kv8Cache c, T* __restrict__ ko, T* __restrict__ vo, const int* __restrict__ base,
                                                       const int* __restrict__ len, int max_len, int* __restrict__ err) {
  chain_enter(ko, vo, base, len, err);
  const int i = blockIdx.y, first = base[i], n = min(len[i], max_len), pk = c.d / V, pv = c.dv / V, per = c.G * (pk + pv);
  const bool ok = n <= 0 || k8_inside(c, first, n);
  if (!ok && blockIdx.x == 0 && threadIdx.x == 0) atomicCAS(err, 0, kK8Place);
  for (long long x = blockIdx.x * 256ll + threadIdx.x; x < (long long)max_len * per; x += gridDim.x * 256ll) {
    const int p = (int)(x / per), y = (int)(x % per);
    const bool is_v = y >= c.G * pk;
    const int z = is_v ? y - c.G * pk : y, pieces = is_v ? pv : pk, width = is_v ? c.dv : c.d, g = z / pieces, at = z % pieces * V;
    float f[V];
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = 0.f;
    if (ok && p < n) {
      const size_t row = (size_t)first + p;
      const int8_t* q = (is_v ? c.v : c.k) + (row * c.G + g) * k8_row(width) + at;
      const float s = (is_v ? c.vs : c.ks)[(row >> c.shift) * c.G + g];
      if (V == 8) {
        const uint2 u = *reinterpret_cast<const uint2*>(q);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)((e < 4 ? u.x : u.y) >> (8 * (e & 3))) * s;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = (float)q[e] * s;
      }
    }
    T* o = (is_v ? vo : ko) + (((size_t)i * max_len + p) * c.G + g) * width + at;
    store_v<V>(o, f);
  }
}

// ---- attention -----------------------------------------------------------------------------------
// All products are integer products of the tensor cores (mma.sync m16n8k32), of the cache's bytes as they are: nothing is converted on
// the way, 23 bytes a clock and SM at the memory's rate.  A query row becomes integers of 23 bits, in units of 2^-21 of its largest
// element's power of two, a weight times its value's scale integers of 23 bits of the largest of 32 of them; each is cut into three bytes,
// which are rows of the left operand, and the three 32-bit sums, exact, join in fp32.  So scores and sums are as good as fp32 ones.
//   rows    groups of 8 (token, head): row r of the operand is the low byte of row r, row r + 8 its middle byte; the high bytes take a
//           second product, whose upper half is empty or another group's
//   keys    lane (g = lane / 4, c = lane % 4) holds bytes 32 c .. 32 c + 31 of key g of 8: the columns may come in any order, the queries' do so too
//   values  the same lane holds columns 16 g .. 16 g + 15 of the keys 8 j + 2 c, 8 j + 2 c + 1 (j < 4), which are those whose scores it has: weights
//           need no exchange, and four keys' bytes of a column come together by byte permutations
//   rings   rows of 128 bytes with TMA's 128-byte swizzle: neither access meets a bank conflict
// The sums start at 12582912 = 1.5 2^23 taken as bits: a sum below 2^22 read as a float is then 12582912 + sum, and a subtraction converts it.
constexpr int kK8Threads = 128, kK8Keys = 32, kK8Stage = 2 * kK8Keys * 128, kK8Stages = 3, kK8Ring = 4 * kK8Stages * kK8Stage;
constexpr int kK8Smem = kK8Ring + 1024;                 // two CTAs an SM, in a split of 196 KB
constexpr int kK8Heads = 16, kK8MaxSplits = 64;
constexpr int kK8Wait = 52;                             // error word: a copy did not arrive
constexpr float kLog2e = 1.4426950408889634f;
static_assert(2 * (kK8Smem + 1024) <= 196 * 1024, "");

struct Kv8Attn {
  Kv8Cache c;
  const void* q;
  void* out;                      // [n, H, dv]
  float* part;                    // [n, H, splits, dv + 2] when splits > 1
  const int *base, *len, *cu;
  const float *sink, *slopes;
  int n, H, ldq, n_seq, tiles, tt, splits, range, window;
  float scale;                    // of the scores, times log2 e 2^-21
  int* err;
};

// The tokens, heads and keys of a CTA: blockIdx.x tile of `tt` tokens of a sequence (cu null: one token each), y: key head and group
// of its query heads, z: range of keys.
struct K8Tile {
  int r0, r1, g, h0, nh, rows, k0, k1, len0, last_first, base;
  __device__ __forceinline__ bool init(const Kv8Attn& a) {
    if (a.cu != nullptr) {
      const int seq = blockIdx.x / a.tiles, end = min(a.cu[seq + 1], a.n);
      r0 = a.cu[seq] + blockIdx.x % a.tiles * a.tt;
      r1 = min(r0 + a.tt, end);
    } else {
      r0 = blockIdx.x;
      r1 = r0 + 1;
    }
    const int rep = a.H / a.c.G, groups = (rep + kK8Heads - 1) / kK8Heads;
    g = blockIdx.y / groups;
    h0 = g * rep + blockIdx.y % groups * kK8Heads;
    nh = min(kK8Heads, (g + 1) * rep - h0);
    if (r0 >= r1) return false;
    rows = (r1 - r0) * nh;
    base = a.base[r0];
    len0 = a.len[r0];
    const int len1 = a.len[r1 - 1];
    k0 = k1 = 0;
    last_first = max(0, len1 - a.window);
    if (len1 > 0) {
      if (!k8_inside(a.c, base, len1)) {
        if (threadIdx.x == 0) atomicCAS(a.err, 0, kK8Place);
      } else {
        k0 = (max(0, len0 - a.window) & ~(kK8Keys - 1)) + (int)blockIdx.z * a.range;
        k1 = min(k0 + a.range, len1);
      }
    }
    return true;
  }
  __device__ __forceinline__ int token(int m) const { return r0 + m / nh; }
  __device__ __forceinline__ int head(int m) const { return h0 + m % nh; }
};

template <typename T>
__device__ __forceinline__ void k8_zero_rows(const Kv8Attn& a, int t0, int h0, int nh) {      // the heads of tokens t0 and on
  T* out = reinterpret_cast<T*>(a.out);
  const long long per = (long long)nh * a.c.dv;
  for (long long i = threadIdx.x; i < (long long)(a.n - t0) * per; i += blockDim.x)
    out[((size_t)(t0 + i / per) * a.H + h0) * a.c.dv + i % per] = from_f<T>(0.f);
}

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
constexpr int kMagic = 0x4b400000;
constexpr float kMagicF = 12582912.f;
// The left operand unsigned, a sum that starts here.
__device__ __forceinline__ void mma_u8_first(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(kMagic));
}
__device__ __forceinline__ float2 k8_sum(int x, int y) { return sm100::fadd2(make_float2(__int_as_float(x), __int_as_float(y)), make_float2(-kMagicF, -kMagicF)); }
// high 2^16 + middle 2^8 + low of two sums
__device__ __forceinline__ float2 k8_join(int l0, int l1, int m0, int m1, int h0, int h1) {
  const float2 b = make_float2(256.f, 256.f);
  return sm100::ffma2(sm100::ffma2(k8_sum(h0, h1), b, k8_sum(m0, m1)), b, k8_sum(l0, l1));
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// Bytes of 4 x 4: x[i] byte j -> x[j] byte i.
__device__ __forceinline__ void transpose_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t (&y)[4]) {
  const uint32_t ab0 = __byte_perm(a, b, 0x5140), ab1 = __byte_perm(a, b, 0x7362), cd0 = __byte_perm(c, d, 0x5140), cd1 = __byte_perm(c, d, 0x7362);
  y[0] = __byte_perm(ab0, cd0, 0x5410);
  y[1] = __byte_perm(ab0, cd0, 0x7632);
  y[2] = __byte_perm(ab1, cd1, 0x5410);
  y[3] = __byte_perm(ab1, cd1, 0x7632);
}

struct K8Ring {
  uint64_t full[4][kK8Stages];    // of a warp's stages
  int gave_up;
};
static_assert(sizeof(K8Ring) <= 128, "");
// The stages start at a multiple of 1024; the barriers lie in what is left in front of them, or behind.
__device__ __forceinline__ uint8_t* k8_stages(uint8_t* raw) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
}
__device__ __forceinline__ K8Ring& k8_ring(uint8_t* raw) {
  uint8_t* stages = k8_stages(raw);
  return *reinterpret_cast<K8Ring*>(stages - raw >= 128 ? raw : stages + kK8Ring);
}

// The 32 elements 32 c .. 32 c + 31 of a row of `d`.
template <typename T>
__device__ __forceinline__ void k8_load_query(const T* src, int c, int d, bool vec, float (&f)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const int at = 32 * c + i;
    float g[8];
    if (vec && at < d) {                                // d a multiple of 8
      load_v<8>(src + at, g);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = at + e < d ? to_f<T>(src[at + e]) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[i + e] = g[e];
  }
}

// What a warp keeps of a group of 8 rows; lane (g, c) has row g.
struct K8Rows {
  uint32_t q[3][4][2];            // bytes of the query: [low, middle, high][32 columns][half]
  float size;                     // power of two of its largest element (NaN where it is not finite)
  float m, l, slope;              // largest score (in powers of two), this lane's share of the sum of the weights
  int first, end;                 // keys the row sees
};
template <typename T>
__device__ __forceinline__ void k8_load_rows(const Kv8Attn& a, const K8Tile& t, int m, int c, K8Rows& r) {
  const int row = min(m, t.rows - 1), tok = t.token(row), h = t.head(row);      // rows past the end repeat the last
  const T* src = reinterpret_cast<const T*>(a.q) + (size_t)tok * a.ldq + (size_t)h * a.c.d;
  const bool vec = a.c.d % 8 == 0 && (reinterpret_cast<uintptr_t>(src) & (8 * sizeof(T) > 16 ? 15 : 8 * sizeof(T) - 1)) == 0;
  float f[32], big = 0.f;
  k8_load_query<T>(src, c, a.c.d, vec, f);
#pragma unroll
  for (int i = 0; i < 32; ++i) big = max_nan(big, fabsf(f[i]));
  big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, 1));
  big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, 2));
  const int e = max((int)(__float_as_uint(big) >> 23), 1);            // biased exponent
  r.size = e >= 255 ? k8_nan() : __uint_as_float((uint32_t)e << 23);
  const float inv = e >= 254 ? __uint_as_float(0x00400000u) : __uint_as_float((uint32_t)(254 - e) << 23);      // 2^-(e - 127)
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint32_t p[3] = {0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int v = __float2int_rn(f[8 * s + 4 * x + i] * inv * 2097152.f);
        const int lo = (int8_t)v, v1 = (v - lo) >> 8, mid = (int8_t)v1, hi = (v1 - mid) >> 8;
        p[0] |= (uint32_t)(lo & 255) << (8 * i);
        p[1] |= (uint32_t)(mid & 255) << (8 * i);
        p[2] |= (uint32_t)(hi & 255) << (8 * i);
      }
#pragma unroll
      for (int y = 0; y < 3; ++y) r.q[y][s][x] = p[y];
    }
  r.end = a.len[tok];
  r.first = max(0, r.end - a.window);
  r.slope = a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.f;
  r.m = -INFINITY;
  r.l = 0.f;
}

// Scales of the keys 8 j + 2 c + e (index 2 j + e) from those of key `lane` a lane.
__device__ __forceinline__ void k8_scales(float mine, int shift, int c, float (&s)[8]) {
  if (shift >= 3) {
#pragma unroll
    for (int j = 0; j < 4; ++j) s[2 * j] = s[2 * j + 1] = __shfl_sync(0xffffffffu, mine, 8 * j);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = __shfl_sync(0xffffffffu, mine, 8 * (i >> 1) + 2 * c + (i & 1));
  }
}

// A group's weights of 32 keys: from scores (integers joined) to bytes.  Returns the factors of the sums before and of these keys'.
struct K8Weights {
  uint32_t p[3][2];               // bytes: [low, middle, high][keys 0 .. 3, 4 .. 7 of the lane]
  float before, now;
};
__device__ __forceinline__ void k8_softmax(const Kv8Attn& a, K8Rows& r, float (&s)[8], const float (&ks)[8], const float (&vs)[8], int key0, int c, bool mask,
                                           K8Weights& w) {
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = s[i] * a.scale * (ks[i] * r.size);
  bool sees[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sees[i] = true;
  if (a.slopes != nullptr || mask) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int key = key0 + 8 * (i >> 1) + 2 * c + (i & 1);
      s[i] = fmaf(r.slope, (float)(key - (r.end - 1)), s[i]);
      sees[i] = key >= r.first && key < r.end;
      if (!sees[i]) s[i] = -INFINITY;
    }
  }
  float mx = sm100::fmax3(sm100::fmax3(s[0], s[1], s[2]), sm100::fmax3(s[3], s[4], s[5]), fmaxf(s[6], s[7]));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  const float now = fmaxf(r.m, mx), ref = now == -INFINITY ? 0.f : now;
  w.before = now == -INFINITY ? 1.f : exp2f(r.m - now);                // no key yet: nothing to rescale
  r.m = now;
  float big = 0.f, sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float p = exp2f(s[i] - ref);
    sum += p;
    s[i] = sees[i] ? p * vs[i] : 0.f;                                  // what a row does not see may have any scale
    big = max_nan(big, s[i]);
  }
  r.l = fmaf(r.l, w.before, sum);
  big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, 1));
  big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, 2));
  const int e = max((int)(__float_as_uint(big) >> 23), 23);            // weights below 2^-104, of values of 10^-32, lose bits
  const float up = __uint_as_float((uint32_t)(276 - min(e, 254)) << 23);                // big up is in 2^22 .. 2^23
  w.now = big != big ? k8_nan() : __uint_as_float((uint32_t)(e - 22) << 23);
  uint32_t f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __float_as_uint(fmaf(s[i], up, 8388608.f));        // the mantissa is the integer
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const uint32_t ab = __byte_perm(f[4 * x], f[4 * x + 1], 0x5140), cd = __byte_perm(f[4 * x + 2], f[4 * x + 3], 0x5140);
    const uint32_t ah = __byte_perm(f[4 * x], f[4 * x + 1], 0x0062), ch = __byte_perm(f[4 * x + 2], f[4 * x + 3], 0x0062);
    w.p[0][x] = __byte_perm(ab, cd, 0x5410);
    w.p[1][x] = __byte_perm(ab, cd, 0x7632);
    w.p[2][x] = __byte_perm(ah, ch, 0x5410);
  }
}

// Scores and weighted values of 32 keys, from `key0` on, in a stage of the ring.  acc: columns 32 c + x and 32 c + 16 + x.
template <int NB>
__device__ __forceinline__ void k8_unit(const Kv8Attn& a, const uint8_t* stage, int key0, bool mask, const float (&ks)[8], const float (&vs)[8], K8Rows (&r)[NB],
                                        float2 (&acc)[NB][16], int gr, int c) {
  float s[NB][8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t k[8];
    const uint8_t* row = stage + (8 * j + gr) * 128;                   // row & 7 = gr
    const uint4 x = *reinterpret_cast<const uint4*>(row + (((2 * c) ^ gr) << 4)), y = *reinterpret_cast<const uint4*>(row + (((2 * c + 1) ^ gr) << 4));
    k[0] = x.x, k[1] = x.y, k[2] = x.z, k[3] = x.w, k[4] = y.x, k[5] = y.y, k[6] = y.z, k[7] = y.w;
    int lm[NB][4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hi[i] = kMagic;
#pragma unroll
      for (int b = 0; b < NB; ++b) lm[b][i] = kMagic;
    }
#pragma unroll
    for (int x4 = 0; x4 < 4; ++x4) {
#pragma unroll
      for (int b = 0; b < NB; ++b) mma_s8(lm[b], r[b].q[0][x4][0], r[b].q[1][x4][0], r[b].q[0][x4][1], r[b].q[1][x4][1], k[2 * x4], k[2 * x4 + 1]);
      mma_s8(hi, r[0].q[2][x4][0], NB == 2 ? r[NB - 1].q[2][x4][0] : 0u, r[0].q[2][x4][1], NB == 2 ? r[NB - 1].q[2][x4][1] : 0u, k[2 * x4], k[2 * x4 + 1]);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const float2 z = k8_join(lm[b][0], lm[b][1], lm[b][2], lm[b][3], hi[2 * b], hi[2 * b + 1]);
      s[b][2 * j] = z.x;
      s[b][2 * j + 1] = z.y;
    }
  }
  K8Weights w[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) k8_softmax(a, r[b], s[b], ks, vs, key0, c, mask, w[b]);
  uint4 v[8];                                                          // 16 columns of this lane's 8 keys
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int key = 8 * (i >> 1) + 2 * c + (i & 1);
    v[i] = *reinterpret_cast<const uint4*>(stage + kK8Keys * 128 + key * 128 + ((gr ^ (2 * c + (i & 1))) << 4));
  }
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    uint32_t b0[4], b1[4], t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = y == 0 ? v[i].x : y == 1 ? v[i].y : y == 2 ? v[i].z : v[i].w;
    transpose_bytes(t[0], t[1], t[2], t[3], b0);
    transpose_bytes(t[4], t[5], t[6], t[7], b1);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      int lm[NB][4], hi[4];
#pragma unroll
      for (int b = 0; b < NB; ++b) mma_u8_first(lm[b], w[b].p[0][0], w[b].p[1][0], w[b].p[0][1], w[b].p[1][1], b0[x], b1[x]);
      mma_u8_first(hi, w[0].p[2][0], NB == 2 ? w[NB - 1].p[2][0] : 0u, w[0].p[2][1], NB == 2 ? w[NB - 1].p[2][1] : 0u, b0[x], b1[x]);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const float2 z = k8_join(lm[b][0], lm[b][1], lm[b][2], lm[b][3], hi[2 * b], hi[2 * b + 1]);
        float2& o = acc[b][4 * y + x];
        o = sm100::ffma2(o, make_float2(w[b].before, w[b].before), make_float2(z.x * w[b].now, z.y * w[b].now));
      }
    }
  }
}

// Few rows: up to 8 NB of them, the keys dealt out to the warps.  A CTA has 4 warps with rings of their own.
template <typename T, int NB>
__global__ void __launch_bounds__(kK8Threads, 2)
attn_kv8_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Kv8Attn a) {
  extern __shared__ __align__(128) uint8_t k8sm_raw[];
  uint8_t* sm = k8_stages(k8sm_raw);
  K8Ring& ring = k8_ring(k8sm_raw);
  if (threadIdx.x == 0) {
    for (int w = 0; w < 4; ++w)
      for (int i = 0; i < kK8Stages; ++i) sm100::mbar_init(&ring.full[w][i], 1);
    sm100::fence_barrier_init();
    sm100::tma_prefetch_desc(&tmK);
    sm100::tma_prefetch_desc(&tmV);
    ring.gave_up = 0;
  }
  __syncthreads();
  chain_enter();
  K8Tile t;
  const bool some = t.init(a);
  if (a.cu != nullptr && blockIdx.x == gridDim.x - 1 && a.splits == 1) k8_zero_rows<T>(a, min(max(a.cu[a.n_seq], 0), a.n), t.h0, t.nh);
  if (!some) return;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, gr = lane >> 2, c = lane & 3;
  uint8_t* stages = sm + warp * kK8Stage * kK8Stages;
  const int units = t.k1 > t.k0 ? (t.k1 - t.k0 + kK8Keys - 1) / kK8Keys : 0, mine = units > warp ? (units - warp + 3) / 4 : 0;
  volatile int* gave_up = &ring.gave_up;
  auto load = [&](int i) {                             // rows past the range are whatever lies there: they are not seen
    if (i < mine && lane == 0) {
      uint8_t* st = stages + i % kK8Stages * kK8Stage;
      uint64_t* bar = &ring.full[warp][i % kK8Stages];
      const int row = t.base + t.k0 + (warp + 4 * i) * kK8Keys;
      sm100::mbar_expect_tx(bar, kK8Stage);
      sm100::tma_load_3d(st, &tmK, bar, 0, t.g, row);
      sm100::tma_load_3d(st + kK8Keys * 128, &tmV, bar, 0, t.g, row);
    }
  };
  float kn[2], vn[2];                                  // scales of key `lane` of the next two units
  auto load_scales = [&](int i, float& k, float& v) {
    if (i < mine) {
      const size_t at = (size_t)((t.base + min(t.k0 + (warp + 4 * i) * kK8Keys + lane, t.k1 - 1)) >> a.c.shift) * a.c.G + t.g;
      k = a.c.ks[at];
      v = a.c.vs[at];
    }
  };
#pragma unroll
  for (int i = 0; i < kK8Stages - 1; ++i) load(i);
  load_scales(0, kn[0], vn[0]);
  load_scales(1, kn[1], vn[1]);
  K8Rows r[NB];
  float2 acc[NB][16];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    k8_load_rows<T>(a, t, b * 8 + gr, c, r[b]);
#pragma unroll
    for (int x = 0; x < 16; ++x) acc[b][x] = make_float2(0.f, 0.f);
  }
  bool failed = false;
  for (int i = 0; i < mine; ++i) {
    float ks[8], vs[8];
    k8_scales(kn[0], a.c.shift, c, ks);
    k8_scales(vn[0], a.c.shift, c, vs);
    kn[0] = kn[1];
    vn[0] = vn[1];
    load_scales(i + 2, kn[1], vn[1]);
    const int stage = i % kK8Stages, key0 = t.k0 + (warp + 4 * i) * kK8Keys;
    failed = !sm100::mbar_wait_warp(&ring.full[warp][stage], (i / kK8Stages) & 1, gave_up);
    if (failed) break;
    load(i + kK8Stages - 1);                           // over the unit before, which all lanes are done with (the fence and the votes)
    k8_unit<NB>(a, stages + stage * kK8Stage, key0, key0 + kK8Keys > min(t.len0, t.k1) || key0 < t.last_first, ks, vs, r, acc, gr, c);
    sm100::fence_proxy_async_smem();                   // these reads before the copies that go over them
    __syncwarp();
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    r[b].l += __shfl_xor_sync(0xffffffffu, r[b].l, 1);
    r[b].l += __shfl_xor_sync(0xffffffffu, r[b].l, 2);
  }
  if (failed) *gave_up = 1;
  __syncthreads();
  if (*gave_up) {                                      // copies in flight land before the CTA ends
    if (threadIdx.x == 0) {
      atomicCAS(a.err, 0, kK8Wait);
      const unsigned long long t0 = sm100::globaltimer_ns();
      while (sm100::globaltimer_ns() - t0 < 200000ull) {
      }
    }
    __syncthreads();
    return;
  }
  // the warps' shares: [warp][row] largest score | sum, then [warp][row][column]
  constexpr int R = 8 * NB, LD = kK8Dim + 4;
  float* stat = reinterpret_cast<float*>(sm);
  float* sums = stat + 8 * R;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int m = warp * R + b * 8 + gr;
    if (c == 0) {
      stat[m] = r[b].m;
      stat[4 * R + m] = r[b].l;
    }
#pragma unroll
    for (int x = 0; x < 16; x += 4) {
      float* o = sums + m * LD + 32 * c + x;
      *reinterpret_cast<float4*>(o) = make_float4(acc[b][x].x, acc[b][x + 1].x, acc[b][x + 2].x, acc[b][x + 3].x);
      *reinterpret_cast<float4*>(o + 16) = make_float4(acc[b][x].y, acc[b][x + 1].y, acc[b][x + 2].y, acc[b][x + 3].y);
    }
  }
  __syncthreads();
  for (int m = warp; m < t.rows; m += 4) {
    float w[4], mx = -INFINITY, l = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) mx = fmaxf(mx, stat[x * R + m]);
    const int h = t.head(m);
    const size_t th = (size_t)t.token(m) * a.H + h;
    const bool last = a.splits == 1;
    const float sk = last && a.sink != nullptr ? a.sink[h] * kLog2e : -INFINITY, top = fmaxf(mx, sk), ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      w[x] = exp2f(stat[x * R + m] - ref);
      l = fmaf(stat[(4 + x) * R + m], w[x], l);
    }
    float* part = nullptr;
    float f = 1.f;
    if (last) {
      const float den = l + exp2f(sk - ref);
      f = den == 0.f ? 0.f : 1.f / den;
    } else {
      part = a.part + (th * a.splits + blockIdx.z) * (a.c.dv + 2);
      if (lane == 0) {
        part[0] = mx;
        part[1] = l;
      }
    }
    for (int x = lane; x < a.c.dv; x += 32) {
      float o = 0.f;
#pragma unroll
      for (int y = 0; y < 4; ++y) o = fmaf(sums[(y * R + m) * LD + x], w[y], o);
      if (last) reinterpret_cast<T*>(a.out)[th * a.c.dv + x] = from_f<T>(o * f);
      else part[2 + x] = o;
    }
  }
}

// A CTA a row and head: joins the ranges.  Those without a key have largest score -inf and sum 0.
template <typename T>
__global__ void __launch_bounds__(kK8Dim) attn_kv8_merge_kernel(const __grid_constant__ Kv8Attn a) {
  chain_enter();
  __shared__ float weight[kK8MaxSplits];
  const int t = blockIdx.x, h = blockIdx.y, step = a.c.dv + 2;
  T* out = reinterpret_cast<T*>(a.out) + ((size_t)t * a.H + h) * a.c.dv;
  if (a.cu != nullptr && t >= a.cu[a.n_seq]) {
    if (threadIdx.x < a.c.dv) out[threadIdx.x] = from_f<T>(0.f);
    return;
  }
  const float* pt = a.part + ((size_t)t * a.H + h) * a.splits * step;
  if (threadIdx.x < 32) {
    const int s0 = threadIdx.x, s1 = threadIdx.x + 32;
    const float m0 = s0 < a.splits ? pt[(size_t)s0 * step] : -INFINITY, m1 = s1 < a.splits ? pt[(size_t)s1 * step] : -INFINITY;
    const float l0 = s0 < a.splits ? pt[(size_t)s0 * step + 1] : 0.f, l1 = s1 < a.splits ? pt[(size_t)s1 * step + 1] : 0.f;
    const float sk = a.sink != nullptr ? a.sink[h] * kLog2e : -INFINITY, top = fmaxf(warp_max(fmaxf(m0, m1)), sk), ref = top == -INFINITY ? 0.f : top;
    const float e0 = exp2f(m0 - ref), e1 = exp2f(m1 - ref), den = warp_sum(l0 * e0 + l1 * e1) + exp2f(sk - ref), f = den == 0.f ? 0.f : 1.f / den;
    weight[s0] = e0 * f;
    weight[s1] = e1 * f;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < a.c.dv; x += kK8Dim) {
    float o = 0.f;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) o = fmaf(pt[(size_t)s * step + 2 + x], weight[s], o);
    out[x] = from_f<T>(o);
  }
}

// How a call runs: tokens of a tile, tiles of a sequence, ranges of keys.
struct K8Plan {
  int tt, tiles, splits, range, nb;
  long long ctas;
};
static K8Plan k8_plan(int n, int n_seq, int max_q, int H, int G, int d, int dv, int max_len, int window) {
  K8Plan p{};
  const int rep = H / G, groups = (rep + kK8Heads - 1) / kK8Heads, nh = std::min(rep, kK8Heads);
  const bool one = n_seq <= 0 || max_q <= 1;
  p.tt = one ? 1 : std::max(1, std::min(max_q, 16 / nh));
  p.tiles = one ? 1 : (max_q + p.tt - 1) / p.tt;
  p.nb = p.tt * nh <= 8 ? 1 : 2;
  p.ctas = (long long)(n_seq > 0 ? (long long)n_seq * p.tiles : n) * G * groups;
  if (window > 0 && max_len > window + p.tt + kK8Keys) max_len = window + p.tt + kK8Keys;      // rows see windows that start apart, ranges at a unit
  max_len = std::max(max_len, 1);
  // Ranges: as many as two CTAs an SM have room for, of 4 units at least.
  const long long most = std::min<long long>((max_len + 4 * kK8Keys - 1) / (4 * kK8Keys), kK8MaxSplits);
  const long long s = std::max<long long>(1, std::min<long long>(most, 2 * kNumSMs / std::max<long long>(1, p.ctas)));
  p.range = (int)(((max_len + s - 1) / s + kK8Keys - 1) / kK8Keys * kK8Keys);
  p.splits = (max_len + p.range - 1) / p.range;
  return p;
}

int make_tmap_bytes_heads(CUtensorMap* map, const void* ptr, uint64_t dim, uint64_t heads, uint64_t rows, uint32_t box_rows);

template <typename T, int NB>
static int launch_attn_kv8(const Kv8Attn& a, const K8Plan& p, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t stream) {
  static bool ready = false;
  if (!ready) {
    const cudaError_t e = cudaFuncSetAttribute(attn_kv8_kernel<T, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, kK8Smem);
    if (e != cudaSuccess) return (int)e;
    ready = true;
  }
  const int groups = (a.H / a.c.G + kK8Heads - 1) / kK8Heads;
  launch_chained(attn_kv8_kernel<T, NB>, dim3(a.cu != nullptr ? a.n_seq * p.tiles : a.n, a.c.G * groups, p.splits), kK8Threads, kK8Smem, stream, tk, tv, a);
  if (p.splits > 1) launch_chained(attn_kv8_merge_kernel<T>, dim3(a.n, a.H), kK8Dim, 0, stream, a);
  return launch_status();
}

static bool k8_sizes_ok(int G, int d, int dv, int shift) {
  return G > 0 && d > 0 && dv > 0 && d <= kK8Dim && dv <= kK8Dim && shift >= 0 && (1 << shift) <= kK8MaxBlock;
}

}  // namespace ell

using namespace ell;

// The rows k [n, G, d], v [n, G, dv] (rows of ldk / ldv elements) of a step: those of cu[i] .. cu[i + 1] - 1 go to the places
// len[cu[i]] - 1 and on of the sequence whose rows start at base[cu[i]].  max_new bounds their number.
ELL_API int ell_kv8_append(int8_t* kc, int8_t* vc, float* ks, float* vs, const void* k, const void* v, const int* base, const int* len, const int* cu,
                           int n, int n_seq, int max_new, int G, int d, int dv, int ldk, int ldv, int shift, long long rows, int is_bf16, int* err,
                           cudaStream_t stream) {
  if (n <= 0 || n_seq <= 0 || max_new <= 0) return 0;
  if (!k8_sizes_ok(G, d, dv, shift)) return -2;
  const Kv8Cache c{kc, vc, ks, vs, rows, G, d, dv, shift};
  const int block = 1 << shift;
  const long long blocks = ((long long)max_new + 2 * block - 2) / block, ctas = ((long long)n_seq * blocks * 2 * G + 7) / 8;
  if (ctas > 0x7fffffff) return -2;
  if (is_bf16)
    launch_chained(kv8_append_kernel<__nv_bfloat16>, (unsigned)ctas, 256, 0, stream, c, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, base, len, cu,
                   n_seq, n, (int)blocks, ldk, ldv, err);
  else
    launch_chained(kv8_append_kernel<float>, (unsigned)ctas, 256, 0, stream, c, (const float*)k, (const float*)v, base, len, cu, n_seq, n, (int)blocks,
                   ldk, ldv, err);
  return launch_status();
}

ELL_API int ell_kv8_read(const int8_t* kc, const int8_t* vc, const float* ks, const float* vs, void* ko, void* vo, const int* base, const int* len,
                         int n, int max_len, int G, int d, int dv, int shift, long long rows, int is_bf16, int* err, cudaStream_t stream) {
  if (n <= 0 || max_len <= 0) return 0;
  if (!k8_sizes_ok(G, d, dv, shift) || n > 65535) return -2;
  const Kv8Cache c{const_cast<int8_t*>(kc), const_cast<int8_t*>(vc), const_cast<float*>(ks), const_cast<float*>(vs), rows, G, d, dv, shift};
  const bool vec = d % 8 == 0 && dv % 8 == 0;
  const dim3 grid(grid_for((long long)max_len * G * (d + dv) / (vec ? 8 : 1), 256, std::max(1, 16 / n)), n);
#define ELL_READ(T, V) launch_chained(kv8_read_kernel<T, V>, grid, 256, 0, stream, c, (T*)ko, (T*)vo, base, len, max_len, err)
  if (is_bf16) vec ? ELL_READ(__nv_bfloat16, 8) : ELL_READ(__nv_bfloat16, 1);
  else vec ? ELL_READ(float, 8) : ELL_READ(float, 1);
#undef ELL_READ
  return launch_status();
}

// Scratch floats a call needs (0: none).  The sizes are those of ell_attn_kv8.
ELL_API long long ell_attn_kv8_scratch(int n, int n_seq, int max_q, int H, int G, int d, int dv, int max_len, int window) {
  if (G <= 0 || H % G) return 0;
  const K8Plan p = k8_plan(n, n_seq, max_q, H, G, d, dv, max_len, window);
  return p.splits == 1 ? 0 : (long long)n * H * p.splits * (dv + 2);
}

// q rows of ldq elements.  max_len bounds len[] (longer rows would be cut).  window: keys a row sees (<= 0: all).  cu [n_seq + 1] (or null): rows
// cu[i] .. cu[i + 1] - 1 are consecutive tokens of one sequence, with one base and lengths that grow by one; max_q bounds their number.
ELL_API int ell_attn_kv8(const void* q, const int8_t* kc, const int8_t* vc, const float* ks, const float* vs, void* out, float* part, const int* base,
                         const int* len, const float* sink, const float* slopes, const int* cu, int n, int n_seq, int max_q, int H, int G, int d, int dv,
                         int ldq, int max_len, int window, float scale, int shift, long long rows, int is_bf16, int* err, cudaStream_t stream) {
  if (n <= 0) return 0;
  if (!k8_sizes_ok(G, d, dv, shift) || H % G || rows > 0x7fffffff || G * ((H / G + kK8Heads - 1) / kK8Heads) > 65535 || H > 65535) return -2;
  if (cu == nullptr) n_seq = 0;
  const K8Plan p = k8_plan(n, n_seq, max_q, H, G, d, dv, max_len, window);
  if (p.splits > 1 && part == nullptr) return -2;
  Kv8Attn a{};
  a.c = Kv8Cache{const_cast<int8_t*>(kc), const_cast<int8_t*>(vc), const_cast<float*>(ks), const_cast<float*>(vs), rows, G, d, dv, shift};
  a.q = q, a.out = out, a.part = part, a.base = base, a.len = len, a.cu = cu, a.sink = sink, a.slopes = slopes;
  a.n = n, a.H = H, a.ldq = ldq, a.n_seq = n_seq, a.tiles = p.tiles, a.tt = p.tt, a.splits = p.splits, a.range = p.range;
  a.window = window > 0 ? window : 0x3fffffff, a.scale = (float)((double)scale * 1.4426950408889634 / 2097152), a.err = err;
  CUtensorMap tk, tv;
  int rc = make_tmap_bytes_heads(&tk, kc, k8_row(d), G, rows, kK8Keys);
  if (!rc) rc = make_tmap_bytes_heads(&tv, vc, k8_row(dv), G, rows, kK8Keys);
  if (rc) return rc;
  if (is_bf16) return p.nb == 1 ? launch_attn_kv8<__nv_bfloat16, 1>(a, p, tk, tv, stream) : launch_attn_kv8<__nv_bfloat16, 2>(a, p, tk, tv, stream);
  return p.nb == 1 ? launch_attn_kv8<float, 1>(a, p, tk, tv, stream) : launch_attn_kv8<float, 2>(a, p, tk, tv, stream);
}
