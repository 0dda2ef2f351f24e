// A key/value cache held in 8 bits: written, read back, attended over.
//
// Rows k [R, G, dk], v [R, G, dv] of int8 (dk, dv: the head sizes rounded up to 16), and a scale for each block of `block` rows
// and head, [R / block, G], fp32.  A scale is a power of two s = 2^e, e >= -126, the least with max|x| <= 127 s (at most 2^121, where
// q is cut to 127: 128 2^121 is past the end of fp32 and bf16); x = q s, |q| <= 127.
// So x / s and q s_old / s are exact but for one rounding to an integer, and q s is exact in bf16 and in fp32: reading back loses
// nothing, and a block that rows join later is off by less than s (s / 2 + s / 4 + ..: a scale that grows at least doubles).
// A block that got a value that is not finite has the scale NaN and reads as NaN.
//
// Every place that comes from the device (a sequence's first row, its length, its tokens' rows) is looked at before it is used: what lies outside
// the cache, or starts inside a block, is neither read nor written, and the error word says so.
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
__device__ __forceinline__ bool k8_inside(const Kv8Cache& c, int base, long long n) {
  return base >= 0 && (base & ((1 << c.shift) - 1)) == 0 && base + n <= c.rows;
}
__device__ __forceinline__ float k8_scale_of(float amax) {       // amax finite, >= 0
  const int e = (int)((__float_as_uint(amax) + 0x1ffffu) >> 23) - 6;      // 127 = 2^6 (2 - 2^-6): carries above that mantissa
  return __uint_as_float((uint32_t)min(max(e, 1), 127 + 121) << 23);
}
__device__ __forceinline__ float k8_nan() { return __int_as_float(0x7fffffff); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// ---- writing -----------------------------------------------------------------------------------
// A warp a block of a sequence, head, and keys or values, heads of a block next to each other.  L lanes a row, V elements each; up to kLoads
// loads are under way together, and a block that fits them stays in registers between its maximum and its bytes.  Rows of the block that
// the step does not bring stay, requantised where the scale grows.  Bound by memory for a prompt and by its chain of loads for a step: 4096 rows of
// 32 heads of 128 (keys and values, 67 MB in, 34 out) 23 us, 4.4 TB/s; 64 rows of 8 heads 4.4 us.  With single elements a lane and the rows read
// again from L2 the first took 80 us; with the elements kept as floats (128 registers a thread, 15 warps an SM) 58.
constexpr float kMagicF = 12582912.f;                             // 1.5 2^23: x + this has round(x) in its low bits
// Low bytes of four words.
__device__ __forceinline__ uint32_t k8_low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
template <bool TOP>
__device__ __forceinline__ uint32_t k8_round(float x, float inv) {      // x inv is exact
  return __float_as_uint(TOP ? fminf(fmaxf(x * inv, -127.f), 127.f) + kMagicF : fmaf(x, inv, kMagicF));
}
template <typename T, int V>
struct K8Elems;
template <>
struct K8Elems<__nv_bfloat16, 8> {
  static constexpr int kLoads = 8;
  uint4 u;
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ float amax(float m) const {
    const uint32_t w[4] = {u.x & 0x7fff7fffu, u.y & 0x7fff7fffu, u.z & 0x7fff7fffu, u.w & 0x7fff7fffu};
    const __nv_bfloat162 a = __hmax2_nan(reinterpret_cast<const __nv_bfloat162&>(w[0]), reinterpret_cast<const __nv_bfloat162&>(w[1]));
    const __nv_bfloat162 b = __hmax2_nan(reinterpret_cast<const __nv_bfloat162&>(w[2]), reinterpret_cast<const __nv_bfloat162&>(w[3]));
    const float2 f = __bfloat1622float2(__hmax2_nan(a, b));
    return max3_nan(m, f.x, f.y);
  }
  template <bool TOP>
  __device__ __forceinline__ void store(int8_t* dst, float inv) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = k8_round<TOP>(__uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16), inv);
    *reinterpret_cast<uint2*>(dst) = make_uint2(k8_low_bytes(r[0], r[1], r[2], r[3]), k8_low_bytes(r[4], r[5], r[6], r[7]));
  }
};
template <>
struct K8Elems<float, 8> {
  static constexpr int kLoads = 4;
  float f[8];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
  }
  __device__ __forceinline__ void load(const float* p) { load_v<8>(p, f); }
  __device__ __forceinline__ float amax(float m) const {
#pragma unroll
    for (int i = 0; i < 8; i += 2) m = max3_nan(m, fabsf(f[i]), fabsf(f[i + 1]));
    return m;
  }
  template <bool TOP>
  __device__ __forceinline__ void store(int8_t* dst, float inv) const {
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = k8_round<TOP>(f[i], inv);
    *reinterpret_cast<uint2*>(dst) = make_uint2(k8_low_bytes(r[0], r[1], r[2], r[3]), k8_low_bytes(r[4], r[5], r[6], r[7]));
  }
};
template <typename T>
struct K8Elems<T, 1> {
  static constexpr int kLoads = 8;
  float f;
  __device__ __forceinline__ void zero() { f = 0.f; }
  __device__ __forceinline__ void load(const T* p) { f = to_f<T>(*p); }
  __device__ __forceinline__ float amax(float m) const { return max_nan(m, fabsf(f)); }
  template <bool TOP>
  __device__ __forceinline__ void store(int8_t* dst, float inv) const { *dst = (int8_t)k8_round<TOP>(f, inv); }
};

template <typename T, int V>
__global__ void __launch_bounds__(256, 4)
kv8_append_kernel(const Kv8Cache c, const T* __restrict__ k, const T* __restrict__ v, const int* __restrict__ base_, const int* __restrict__ len_,
                  const int* __restrict__ cu, int n, int blocks, int ldk, int ldv, int* __restrict__ err) {
  chain_enter(k, v, base_, len_, cu, err);
  const unsigned wide = 2u * c.G, across = (wide + 7) / 8, j = blockIdx.x / across, item = (blockIdx.x - j * across) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, which = item >= (unsigned)c.G, g = (int)item - which * c.G, s = blockIdx.y;
  if (item >= wide) return;
  const int r0 = cu[s], count = min(cu[s + 1], n) - r0;
  if (count <= 0 || r0 < 0) return;
  const int base = base_[r0], p0 = len_[r0] - 1;
  if (p0 < 0) return;                                             // padding
  if (!k8_inside(c, base, (long long)p0 + count)) {
    if (lane == 0) atomicCAS(err, 0, kK8Place);
    return;
  }
  const int b = (p0 >> c.shift) + (int)j, start = b << c.shift, first = max(p0, start), last = min(p0 + count, start + (1 << c.shift));
  if (first >= last) return;
  if (lane == 0 && (int)j == blocks - 1 && last < p0 + count) atomicCAS(err, 0, kK8Place);      // more rows than was said: they are left out
  const int width = which ? c.dv : c.d, row = k8_row(width), step = c.G * row, rows = last - first;
  const size_t ld = which ? ldv : ldk;
  const T* src = (which ? v : k) + (size_t)(r0 + first - p0) * ld + (size_t)g * width;
  float* scale = (which ? c.vs : c.ks) + ((size_t)(base >> c.shift) + b) * c.G + g;
  const float old = first > start ? *scale : 0.f;
  int8_t* dst = (which ? c.v : c.k) + ((size_t)base * c.G + g) * row;
  int shift = 0;                                                  // lanes of a row: a power of two
  while ((V << shift) < row && shift < 5) ++shift;
  const int per = 32 >> shift, my_row = lane >> shift, piece = lane & ((1 << shift) - 1);
  constexpr int kLoads = K8Elems<T, V>::kLoads;
  const int turns = V == 1 ? (row + 31) / 32 : 1, chunk = per * kLoads;      // single elements of a row take several turns
  const bool kept = rows <= chunk && turns == 1;
  K8Elems<T, V> e[kLoads];
  auto load = [&](int at, int r) {
    const T* from = src + (size_t)(r + my_row) * ld + at;
    const int mine = at < width ? rows - r - my_row : 0;          // rows of this lane, one of `per`
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      e[i].zero();
      if (i * per < mine) e[i].load(from + (size_t)(i * per) * ld);
    }
  };
  float amax = 0.f;
  for (int x = 0; x < turns; ++x)
    for (int r = 0; r < rows; r += chunk) {
      load(x * 32 + piece * V, r);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) amax = e[i].amax(amax);
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  float now = amax <= 3.4028235e38f ? k8_scale_of(amax) : k8_nan();
  if (first > start) {                                            // rows that were there
    const bool grows = !(old >= now);
    if (old != old) now = old;
    else if (!grows) now = old;
    if (grows && now == now) {
      const float ratio = old / now;
      for (int p = start; p < first; ++p)
        for (int x = lane * 4; x < row; x += 128) {
          uint32_t* q = reinterpret_cast<uint32_t*>(dst + (size_t)p * step + x);
          const uint32_t w = *q;
          uint32_t z[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) z[i] = k8_round<false>((float)(int8_t)(w >> (8 * i)), ratio);
          *q = k8_low_bytes(z[0], z[1], z[2], z[3]);
        }
    }
  }
  const bool none = now != now, top = now == k8_scale_of(3.4028235e38f);
  const float inv = none ? 0.f : __uint_as_float(0x7f000000u - __float_as_uint(now));      // of a power of two
  for (int x = 0; x < turns; ++x)
    for (int r = 0; r < rows; r += chunk) {
      const int at = x * 32 + piece * V;
      if (!kept) load(at, r);
      if (none) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) e[i].zero();
      }
      int8_t* to = dst + (size_t)(first + r + my_row) * step + at;
      const int mine = at < row ? rows - r - my_row : 0;          // rows of this lane, one of `per`
      if (top) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          if (i * per < mine) e[i].template store<true>(to + (size_t)(i * per) * step, inv);
      } else {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          if (i * per < mine) e[i].template store<false>(to + (size_t)(i * per) * step, inv);
      }
    }
  __syncwarp();                                                   // everybody has read the old scale
  if (lane == 0) *scale = now;
}

// ---- reading back ------------------------------------------------------------------------------
// Bytes times a scale: a byte and 128 is put into the mantissa of 2^23, from which 2^23 + 128 is taken (an integer's own conversion has a
// quarter of this rate).  The products are exact in bf16 too: their upper halves.
template <int V, typename T>
__device__ __forceinline__ void k8_store_values(T* o, const uint32_t* w, float s) {
  constexpr bool kHalf = sizeof(T) == 2;
  if (V == 8) {
    float2 f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = w[i / 2] ^ 0x80808080u;
      f[i] = make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, i & 1 ? 0x7552 : 0x7550)),
                         __uint_as_float(__byte_perm(u, 0x4b000000u, i & 1 ? 0x7553 : 0x7551)));
      f[i] = sm100::fmul2(sm100::fadd2(f[i], make_float2(-8388736.f, -8388736.f)), make_float2(s, s));
    }
    if (kHalf) {
      uint4 z;
      z.x = __byte_perm(__float_as_uint(f[0].x), __float_as_uint(f[0].y), 0x7632);
      z.y = __byte_perm(__float_as_uint(f[1].x), __float_as_uint(f[1].y), 0x7632);
      z.z = __byte_perm(__float_as_uint(f[2].x), __float_as_uint(f[2].y), 0x7632);
      z.w = __byte_perm(__float_as_uint(f[3].x), __float_as_uint(f[3].y), 0x7632);
      *reinterpret_cast<uint4*>(o) = z;
    } else {
      reinterpret_cast<float4*>(o)[0] = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
      reinterpret_cast<float4*>(o)[1] = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
    }
  } else {
    *o = from_f<T>((float)(int8_t)w[0] * s);
  }
}
// ko [n, max_len, G, d], vo [n, max_len, G, dv].  cu null: rows base[i] .. base[i] + len[i] - 1 of the cache, then zeros.  Otherwise sequence i has
// the query rows cu[i] .. cu[i + 1] - 1 with base and len of their own: its rows are those that its last one sees, nothing is written behind them,
// row_base[r] becomes the place of a query row's keys in ko, row_base[rows + r] its length, max_len at most; both are 0 for rows behind the
// last sequence.  A thread keeps its place in a row, V elements, and takes positions, eight of which are under way together.
// Bound by memory: 8 prefixes of up to 4096 rows, 8 heads of 128 (37 MB
// in, 134 MB out, zeros among them) 30 us among others, 5.7 TB/s, 35 alone with a cold L2.  With a division for every eight values it took
// 48 us, with conversions of the integers 39, with 16 values a thread, whose stores leave every other 16 bytes to the next one, 134.  One
// prompt of 4096 rows of 32 heads 18.5 us; 27 where a CTA took four positions of whole rows.
template <typename T, int V>
__global__ void __launch_bounds__(256, 4)
kv8_read_kernel(const Kv8Cache c, T* __restrict__ ko, T* __restrict__ vo, const int* __restrict__ base, const int* __restrict__ len,
                const int* __restrict__ cu, int* __restrict__ row_base, int rows, int max_len, int chunk, int* __restrict__ err) {
  chain_enter(ko, vo, base, len, cu, row_base, err);
  const int i = blockIdx.y, pk = c.d / V, pv = c.dv / V, per = c.G * (pk + pv);
  int r0 = i, r1 = i + 1;
  if (cu != nullptr) {
    r0 = cu[i];
    r1 = min(cu[i + 1], rows);
    if (i == gridDim.y - 1 && blockIdx.x == 0 && blockIdx.z == 0)
      for (int r = max(r1, 0) + threadIdx.x; r < rows; r += 256) row_base[r] = row_base[rows + r] = 0;
    if (r0 < 0 || r0 >= r1) return;
    if (blockIdx.x == 0 && blockIdx.z == 0)
      for (int r = r0 + threadIdx.x; r < r1; r += 256) {
        row_base[r] = i * max_len;
        row_base[rows + r] = min(len[r], max_len);
      }
  }
  const int first = base[r0], n = min(len[r1 - 1], max_len);
  const bool ok = n <= 0 || k8_inside(c, first, n);
  if ((!ok || (cu != nullptr && len[r1 - 1] > max_len)) && blockIdx.x == 0 && threadIdx.x == 0) atomicCAS(err, 0, kK8Place);
  const int p0 = blockIdx.x * chunk, p1 = min(p0 + chunk, cu != nullptr && ok ? n : max_len);
  const int beside = max(1, 256 / per);                          // positions that the threads take side by side
  const int y = blockIdx.z * 256 + threadIdx.x;
  if (y < beside * per) {
    const int z0 = y % per, at_p = y / per;
    const bool is_v = z0 >= c.G * pk;
    const int z = is_v ? z0 - c.G * pk : z0, pieces = is_v ? pv : pk, width = is_v ? c.dv : c.d, row = k8_row(width);
    const int g = z / pieces, at = z % pieces * V;
    const int step = c.G * row, out_step = c.G * width, mine = ok ? min(n, p1) : 0;
    const int8_t* q = (is_v ? c.v : c.k) + ((size_t)first * c.G + g) * row + at;
    const float* scale = (is_v ? c.vs : c.ks) + (size_t)(first >> c.shift) * c.G + g;
    T* o = (is_v ? vo : ko) + ((size_t)i * max_len * c.G + g) * width + at;
    constexpr int kLoads = V == 8 ? 8 : 4;
    int p = p0 + at_p;
    for (; p < mine; p += kLoads * beside) {
      uint32_t w[kLoads][V == 8 ? 2 : 1];
      float s[kLoads];
#pragma unroll
      for (int x = 0; x < kLoads; ++x) {
        const int r = min(p + x * beside, mine - 1);
        s[x] = scale[(size_t)(r >> c.shift) * c.G];
        if (V == 8) {
          const uint2 u = *reinterpret_cast<const uint2*>(q + (size_t)r * step);
          w[x][0] = u.x;
          w[x][V == 8] = u.y;
        } else {
          w[x][0] = (uint8_t)q[(size_t)r * step];
        }
      }
#pragma unroll
      for (int x = 0; x < kLoads; ++x)
        if (p + x * beside < mine) k8_store_values<V>(o + (size_t)(p + x * beside) * out_step, w[x], s[x]);
    }
    for (p = max(p0, (mine - p0 - at_p + beside - 1) / beside * beside + p0) + at_p; p < p1; p += beside) {      // behind the sequence
      const float none[V] = {};
      store_v<V>(o + (size_t)p * out_step, none);
    }
  }
}

// Rows that see nothing, and those behind the last sequence, of out [n, width]: zero.
__global__ void __launch_bounds__(256)
kv8_clear_kernel(__nv_bfloat16* __restrict__ out, const int* __restrict__ len, const int* __restrict__ cu, int n_seq, int n, int width) {
  chain_enter(out, len, cu);
  const int end = cu[n_seq];
  for (int t = blockIdx.x * 8 + (threadIdx.x >> 5); t < n; t += gridDim.x * 8)
    if (t >= end || len[t] <= 0)
      for (int x = threadIdx.x & 31; x < width; x += 32) out[(size_t)t * width + x] = __float2bfloat16_rn(0.f);
}

// ---- attention -----------------------------------------------------------------------------------
// All products are integer products of the tensor cores (mma.sync m16n8k32), of the cache's bytes as they are: nothing is converted on
// the way, 23 bytes a clock and SM at the memory's rate.  A query row becomes integers of 23 bits, in units of 2^-21 of its largest
// element's power of two, a weight times its value's scale integers of 23 bits of the largest of 64 of them; each is cut into three bytes,
// which are rows of the left operand, and the three 32-bit sums, exact, join in fp32.  So scores and sums are as good as fp32 ones where a row's
// elements are of one size (4e-7 to 8e-7 off 64 bits in the norm, as fp32 sums are); one that is 2^k below its row's largest has k bits less.
//   rows    groups of 8 (token, head): row r of the operand is the low byte of row r, row r + 8 its middle byte; the high bytes take a
//           second product, whose upper half is empty or another group's
//   keys    lane (g = lane / 4, c = lane % 4) holds bytes 32 c .. 32 c + 31 of key g of 8: the columns may come in any order, the queries' do so too
//   values  the same lane holds columns 16 g .. 16 g + 15 of the keys 8 j + 2 c, 8 j + 2 c + 1 (j < 8), which are those whose scores it has: weights
//           need no exchange, and four keys' bytes of a column come together by byte permutations
//   rings   rows of 128 bytes with TMA's 128-byte swizzle: neither access meets a bank conflict
// Bound by memory where sequences are long, by what begins and ends a call (3 us until the first copy, 5 for the join) where they are short.
// Bytes of the cache a second, and us beside those of attention over the same cache in 16 bits: 64 sequences of up to 8192 keys, 32 heads
// on 8, 5.3 to 5.6 TB/s by the GPU, 98 to 105 (216); 24 of up to 4096, 32 on 32, 4.9 to 5.4, 78 to 86 (149); one of 131071, 64 on 8, 4.7, 58
// (92); 6 of up to 1900 with 5 tokens each, 40 on 40, 2.5, 27 (52); one of 203 keys 5.5 (5.6) in a chain of calls, 10.2 (10.2) alone with a
// cold L2: there the cache's size counts for nothing.  Two groups of rows (NB = 2) take 255 registers and spill 80 bytes.
// Steps, us of the first two: a warp a row on the fp32 units 8398 and 4193; integer products with 32 keys a step, a CTA an item 153 and 103;
// equal shares, 64 keys a step 119 and 100; found and joined with fewer barriers 110 and 91; two CTAs an SM with three stages in place of
// three with two 105 and 86; items' beginnings counted 103 and 85.
constexpr int kK8Threads = 128, kK8Keys = 64, kK8Stage = kK8Keys * 128;       // a stage: keys, or values
// Stages of a warp and CTAs an SM, which are to fit a split of 196 KB with the system's 1 KB each (112 bytes more take 228 KB, which later
// kernels find their L1 cut down by).
template <int NB>
struct K8Ring {
  static constexpr int kStages = 3, kCtas = 2, kBytes = 4 * kStages * kK8Stage;
  uint64_t full[4][kStages];
  int gave_up, free_stage[4];
  int piece[4];                   // of the current piece: first token, rows, where it begins, quanta behind its end
  // A warp's sums of a piece go through one stage, [row][column], largest scores and sums of weights behind them or here.
  static constexpr int kRows = 8 * NB, kSumBytes = kRows * kK8Dim * 4;
  static constexpr bool kStatHere = kSumBytes + kRows * 8 > kK8Stage;
  float2 stat[kStatHere ? 4 * kRows : 1];
};
template <int NB>
constexpr int k8_smem() { return K8Ring<NB>::kBytes + (int)sizeof(K8Ring<NB>); }
template <int NB>
constexpr bool k8_fits() { return K8Ring<NB>::kSumBytes <= kK8Stage && K8Ring<NB>::kCtas * (k8_smem<NB>() + 1024) <= 196 * 1024; }
static_assert(k8_fits<1>() && k8_fits<2>(), "");
// Place of columns 4 i .. 4 i + 3 of row m: the lanes that write a row's or several rows' columns together meet in no bank.
__device__ __forceinline__ int k8_sum_at(int m, int i) { return m * kK8Dim + 4 * (i ^ (((m & 7) ^ (2 * (i >> 3))) & 7)); }
constexpr int kK8Heads = 16;
constexpr int kK8Wait = 52;                             // error word: a copy did not arrive
constexpr float kLog2e = 1.4426950408889634f;

struct Kv8Attn {
  Kv8Cache c;
  const void* q;
  void* out;                      // [n, H, dv]
  float* part;                    // when shares are cut: two slots a CTA, then the CTAs' K8Cut
  const int *base, *len, *cu;
  const float *sink, *slopes;
  int n, H, ldq, n_seq, tiles, tt, cut, window, max_len;
  float scale;                    // of the scores, times log2 e 2^-21
  int* err;
};
__host__ __device__ __forceinline__ int k8_groups(int H, int G) { return G * ((H / G + kK8Heads - 1) / kK8Heads); }

// Work is counted in quanta of 256 keys, one unit of 64 for each warp of a CTA.  An item is a tile of `tt` tokens of a sequence (cu null: one
// token) with the query heads of a key head, at most 16 of them.  To begin an item costs a CTA as much as a quantum (queries, sums; 64
// sequences of up to 8192 keys took 105.5 us without that in the shares, 103 with it).
constexpr int kK8Quantum = 4 * kK8Keys;
struct K8Tile {
  int r0, r1, base, len0, len1, low;              // low: where its keys begin, at a unit
  __device__ __forceinline__ K8Tile(const Kv8Attn& a, int x) {
    r0 = x;
    r1 = x + 1;
    if (a.cu != nullptr) {
      const int seq = x / a.tiles, end = min(a.cu[seq + 1], a.n);
      r0 = a.cu[seq] + x % a.tiles * a.tt;
      r1 = min(r0 + a.tt, end);
    }
    len0 = len1 = low = base = 0;
    if (r0 < 0) r1 = r0;
    if (r0 >= r1) return;
    if (a.cu != nullptr && x % a.tiles == a.tiles - 1 && r1 < min(a.cu[x / a.tiles + 1], a.n))
      atomicCAS(a.err, 0, kK8Place);                   // more tokens than was said
    len0 = a.len[r0];
    len1 = a.len[r1 - 1];
    base = a.base[r0];
    const bool in = len1 <= 0 || k8_inside(a.c, base, len1);
    if (!in || len1 > a.max_len) atomicCAS(a.err, 0, kK8Place);        // a longer sequence than was said is answered all the same
    if (!in) len1 = 0;
    len1 = max(len1, 0);
    len0 = min(max(len0, 0), len1);
    low = max(0, len0 - a.window) & ~(kK8Keys - 1);
  }
  __device__ __forceinline__ int quanta() const { return r0 >= r1 ? 0 : max(1, (len1 - low + kK8Quantum - 1) / kK8Quantum); }
  __device__ __forceinline__ int cost() const { return r0 >= r1 ? 0 : quanta() + 1; }
};
// What a CTA does at a time: quanta q0 .. q1 - 1 of a tile.  From places in the tile's cost, of which the first is its beginning.
struct K8Piece {
  K8Tile t;
  int q0, q1, quanta, behind;      // behind: cost of what is left of the tile
  __device__ __forceinline__ K8Piece(const Kv8Attn& a, int x, int q0_, int most) : t(a, x) {
    quanta = t.quanta();
    const int end = min(t.cost(), q0_ + most);
    behind = t.cost() - end;
    q0 = max(0, q0_ - 1);
    q1 = max(0, end - 1);
  }
  __device__ __forceinline__ int k0() const { return t.low + q0 * kK8Quantum; }
  __device__ __forceinline__ int k1() const { return min(t.low + q1 * kK8Quantum, t.len1); }
  __device__ __forceinline__ int units(int warp) const { return max(0, (k1() - k0() - warp * kK8Keys + kK8Quantum - 1) / kK8Quantum); }
};
// The next tile with rows, or n_x.
__device__ __forceinline__ int k8_next(const Kv8Attn& a, int n_x, int x) {
  while (++x < n_x)
    if (a.cu == nullptr || (a.cu[x / a.tiles] >= 0 && a.cu[x / a.tiles] + x % a.tiles * a.tt < min(a.cu[x / a.tiles + 1], a.n))) break;
  return x;
}
// Where share i of n begins among `all` quanta.
__device__ __forceinline__ int k8_share(int i, int all, int n) {
  // shares are below 2^12, as CTAs that are resident are
  return all < (1 << 20) ? (int)((unsigned)i * (unsigned)all / (unsigned)n) : (int)((long long)i * all / n);
}
// What the joining kernel needs to know of an item that begins in a CTA's share and is cut by its end.
struct K8Cut {
  int r0, rows, h0, nh, more;     // more: shares after this one that have a piece of it (0: nothing was cut)
};
constexpr int kK8SlotRow = kK8Dim + 4;            // floats of a row in a slot: sums | largest score, sum of weights

// Columns 4 lane .. 4 lane + 3 of a head's output.
template <typename T>
__device__ __forceinline__ void k8_store_row(const Kv8Attn& a, int tok, int h, int lane, float4 o) {
  T* out = reinterpret_cast<T*>(a.out) + ((size_t)tok * a.H + h) * a.c.dv + 4 * lane;
  const float f[4] = {o.x, o.y, o.z, o.w};
  if (a.c.dv % 4 == 0) {
    if (4 * lane < a.c.dv) store_v<4>(out, f);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * lane + i < a.c.dv) out[i] = from_f<T>(f[i]);
  }
}

// The sums start at 12582912 = 1.5 2^23 taken as bits: a sum below 2^22 read as a float is then 12582912 + sum, and a subtraction converts it.
constexpr uint32_t kMagic = 0x4b400000;
// The left operand signed (queries) or not (weights).  `first`: a sum that starts here, from `zero`.
template <bool SIGNED>
__device__ __forceinline__ void mma_i8(int (&c)[4], bool first, const uint32_t (&zero)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
#define ELL_MMA(TYPE)                                                                                                                  \
  if (first)                                                                                                                           \
    asm("mma.sync.aligned.m16n8k32.row.col.s32." TYPE ".s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"    \
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])                                                                               \
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(zero[0]), "r"(zero[1]), "r"(zero[2]), "r"(zero[3]));       \
  else                                                                                                                                 \
    asm("mma.sync.aligned.m16n8k32.row.col.s32." TYPE ".s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"        \
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])                                                                               \
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  if (SIGNED) {
    ELL_MMA("s8")
  } else {
    ELL_MMA("u8")
  }
#undef ELL_MMA
}
// A constant that the compiler takes for a variable, so that it is kept in a register instead of made again wherever it is used: an
// operand of four registers is then put together once.
__device__ __forceinline__ uint32_t k8_kept(uint32_t x) {
  uint32_t y;
  asm volatile("shfl.sync.idx.b32 %0, %1, 0, 31, 0xffffffff;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float2 k8_sum(int x, int y) {
  return sm100::fadd2(make_float2(__int_as_float(x), __int_as_float(y)), make_float2(-kMagicF, -kMagicF));
}
// high 2^16 + middle 2^8 + low of two sums
__device__ __forceinline__ float2 k8_join(int l0, int l1, int m0, int m1, int h0, int h1) {
  const float2 b = make_float2(256.f, 256.f);
  return sm100::ffma2(sm100::ffma2(k8_sum(h0, h1), b, k8_sum(m0, m1)), b, k8_sum(l0, l1));
}
// Bytes of 4 x 4: x[i] byte j -> x[j] byte i.
__device__ __forceinline__ void transpose_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t (&y)[4]) {
  const uint32_t ab0 = __byte_perm(a, b, 0x5140), ab1 = __byte_perm(a, b, 0x7362), cd0 = __byte_perm(c, d, 0x5140), cd1 = __byte_perm(c, d, 0x7362);
  y[0] = __byte_perm(ab0, cd0, 0x5410);
  y[1] = __byte_perm(ab0, cd0, 0x7632);
  y[2] = __byte_perm(ab1, cd1, 0x5410);
  y[3] = __byte_perm(ab1, cd1, 0x7632);
}

// The 32 elements 32 c .. 32 c + 31 of a query row, as they come, with what else a row of queries needs from memory: all of it is asked for
// before any of it is looked at.
template <typename T>
struct K8Query {
  static constexpr int kWords = 8 * sizeof(T);         // of 32 elements
  uint32_t u[kWords];
  float slope;
  int end;
  __device__ __forceinline__ void load(const Kv8Attn& a, int tok, int h, int c) {
    const T* src = reinterpret_cast<const T*>(a.q) + (size_t)tok * a.ldq + (size_t)h * a.c.d + 32 * c;
    const int d = a.c.d - 32 * c;
    if (a.c.d % 8 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const bool in = i * 4 / (int)sizeof(T) < d;
        const uint4 w = in ? *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(src) + i) : make_uint4(0, 0, 0, 0);
        u[i] = w.x, u[i + 1] = w.y, u[i + 2] = w.z, u[i + 3] = w.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float f = i < d ? to_f<T>(src[i]) : 0.f;
        if (sizeof(T) == 4) u[i % kWords] = __float_as_uint(f);
        else u[i / 2 % kWords] = i & 1 ? u[i / 2 % kWords] | (__float_as_uint(f) & 0xffff0000u) : __float_as_uint(f) >> 16;
      }
    }
    end = a.len[tok];
    slope = a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.f;
  }
  __device__ __forceinline__ float at(int i) const {
    if (sizeof(T) == 4) return __uint_as_float(u[i % kWords]);
    return __uint_as_float(i & 1 ? u[i / 2 % kWords] & 0xffff0000u : u[i / 2 % kWords] << 16);
  }
};
// What a warp keeps of a group of 8 rows; lane (g, c) has row g.
struct K8Rows {
  uint32_t q[4][4], high[4][2];   // bytes of the query, of 32 columns each: low and middle as an operand, high
  float size;                     // power of two of its largest element (NaN where it is not finite)
  float m, l, slope;              // largest score (in powers of two), this lane's share of the sum of the weights
  int first, end;                 // keys the row sees
};
template <typename T>
__device__ __forceinline__ void k8_rows(const Kv8Attn& a, const K8Query<T>& f, K8Rows& r) {
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < 32; i += 2) big = max3_nan(big, fabsf(f.at(i)), fabsf(f.at(i + 1)));
  big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, 1));
  big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, 2));
  const int e = max((int)(__float_as_uint(big) >> 23), 1);            // biased exponent
  r.size = e >= 255 ? k8_nan() : __uint_as_float((uint32_t)e << 23);
  const float inv = e >= 254 ? __uint_as_float(0x00400000u) : __uint_as_float((uint32_t)(254 - e) << 23);      // 2^-(e - 127)
  // v + 0x808080 has the three signed digits of v in its bytes, plus 128 each
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint32_t v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (__float_as_uint(fmaf(f.at(8 * s + 4 * x + i) * inv, 2097152.f, kMagicF)) - kMagic + 0x808080u) ^ 0x808080u;
      const uint32_t ab = __byte_perm(v[0], v[1], 0x5140), cd = __byte_perm(v[2], v[3], 0x5140);
      r.q[s][2 * x] = __byte_perm(ab, cd, 0x5410);
      r.q[s][2 * x + 1] = __byte_perm(ab, cd, 0x7632);
      r.high[s][x] = __byte_perm(__byte_perm(v[0], v[1], 0x0062), __byte_perm(v[2], v[3], 0x0062), 0x5410);
    }
  r.end = f.end;
  r.first = max(0, r.end - a.window);
  r.slope = f.slope;
  r.m = -INFINITY;
  r.l = 0.f;
}

// Scales of the keys 8 j + 2 c + e (index 2 j + e) from those of keys `lane` and lane + 32 a lane.
__device__ __forceinline__ void k8_scales(const float (&mine)[2], int shift, int c, float (&s)[16]) {
  if (shift >= 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) s[4 * j] = s[4 * j + 1] = s[4 * j + 2] = s[4 * j + 3] = __shfl_sync(0xffffffffu, mine[j >> 1], 16 * (j & 1));
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __shfl_sync(0xffffffffu, mine[i >> 3], 8 * ((i >> 1) & 3) + 2 * c + (i & 1));
  }
}

// A group's weights of 64 keys: from scores (integers joined) to bytes.  With the factors of the sums before and of these keys'.
struct K8Weights {
  uint32_t p[2][4], high[2][2];   // bytes, of 32 keys each: low and middle as an operand, high
  float before, now;
};
__device__ __forceinline__ void k8_softmax(const Kv8Attn& a, K8Rows& r, float (&s)[16], const float (&ks)[16], const float (&vs)[16], int key0,
                                           int c, bool mask, K8Weights& w) {
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const float2 f = sm100::fmul2(make_float2(ks[i], ks[i + 1]), make_float2(r.size, r.size));
    const float2 z = sm100::fmul2(sm100::fmul2(make_float2(s[i], s[i + 1]), make_float2(a.scale, a.scale)), f);
    s[i] = z.x;
    s[i + 1] = z.y;
  }
  uint32_t hidden = 0;
  if (a.slopes != nullptr || mask) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = key0 + 8 * (i >> 1) + 2 * c + (i & 1);
      s[i] = fmaf(r.slope, (float)(key - (r.end - 1)), s[i]);
      if (key < r.first || key >= r.end) {
        s[i] = -INFINITY;
        hidden |= 1u << i;
      }
    }
  }
  float mx = fmaxf(s[0], s[1]);
#pragma unroll
  for (int i = 2; i < 16; i += 2) mx = sm100::fmax3(mx, s[i], s[i + 1]);
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  const float now = fmaxf(r.m, mx), ref = now == -INFINITY ? 0.f : now;
  w.before = now == -INFINITY ? 1.f : exp2f(r.m - now);                // no key yet: nothing to rescale
  r.m = now;
  float2 sum = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    float2 z = sm100::fadd2(make_float2(s[i], s[i + 1]), make_float2(-ref, -ref));
    z = make_float2(exp2f(z.x), exp2f(z.y));
    sum = sm100::fadd2(sum, z);
    z = sm100::fmul2(z, make_float2(vs[i], vs[i + 1]));
    s[i] = z.x;
    s[i + 1] = z.y;
  }
  r.l = fmaf(r.l, w.before, sum.x + sum.y);
  if (mask) {                                                          // what a row does not see may have any scale
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (hidden >> i & 1) s[i] = 0.f;
  }
  float big = max_nan(s[0], s[1]);
#pragma unroll
  for (int i = 2; i < 16; i += 2) big = max3_nan(big, s[i], s[i + 1]);
  big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, 1));
  big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, 2));
  const int e = max((int)(__float_as_uint(big) >> 23), 23);            // weights below 2^-104, of values of 10^-32, lose bits
  const float up = __uint_as_float((uint32_t)(276 - min(e, 254)) << 23);                // big up is in 2^22 .. 2^23
  w.now = big != big ? k8_nan() : __uint_as_float((uint32_t)(e - 22) << 23);
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    uint32_t f[4];
#pragma unroll
    for (int i = 0; i < 4; i += 2) {                                   // the mantissa is the integer
      const float2 z = sm100::ffma2(make_float2(s[4 * x + i], s[4 * x + i + 1]), make_float2(up, up), make_float2(8388608.f, 8388608.f));
      f[i] = __float_as_uint(z.x);
      f[i + 1] = __float_as_uint(z.y);
    }
    const uint32_t ab = __byte_perm(f[0], f[1], 0x5140), cd = __byte_perm(f[2], f[3], 0x5140);
    const uint32_t ah = __byte_perm(f[0], f[1], 0x0062), ch = __byte_perm(f[2], f[3], 0x0062);
    w.p[x >> 1][2 * (x & 1)] = __byte_perm(ab, cd, 0x5410);
    w.p[x >> 1][2 * (x & 1) + 1] = __byte_perm(ab, cd, 0x7632);
    w.high[x >> 1][x & 1] = __byte_perm(ah, ch, 0x5410);
  }
}

// Scores of 64 keys in a stage of the ring, as joined integers.
template <int NB>
__device__ __forceinline__ void k8_scores(const uint8_t* stage, const K8Rows (&r)[NB], const uint32_t (&high)[4][4], const uint32_t (&zero)[4],
                                          float (&s)[NB][16], int gr, int c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint32_t k[8];
    const uint8_t* row = stage + (8 * j + gr) * 128;                   // row & 7 = gr
    const uint4 x = *reinterpret_cast<const uint4*>(row + (((2 * c) ^ gr) << 4));
    const uint4 y = *reinterpret_cast<const uint4*>(row + (((2 * c + 1) ^ gr) << 4));
    k[0] = x.x, k[1] = x.y, k[2] = x.z, k[3] = x.w, k[4] = y.x, k[5] = y.y, k[6] = y.z, k[7] = y.w;
    int lm[NB][4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int b = 0; b < NB; ++b) mma_i8<true>(lm[b], i == 0, zero, r[b].q[i], k[2 * i], k[2 * i + 1]);
      mma_i8<true>(hi, i == 0, zero, high[i], k[2 * i], k[2 * i + 1]);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const float2 z = k8_join(lm[b][0], lm[b][1], lm[b][2], lm[b][3], hi[2 * b], hi[2 * b + 1]);
      s[b][2 * j] = z.x;
      s[b][2 * j + 1] = z.y;
    }
  }
}

// Adds 64 keys' weighted values.  A lane reads columns 16 g + 8 (half ^ (g >> 1 & 1)) .. of its keys at a time, so that no two lanes meet
// in a bank; acc[8 half + x] are columns 32 c + 8 (half ^ (c & 1)) + x and that + 16.
template <int NB>
__device__ __forceinline__ void k8_values(const uint8_t* stage, const K8Weights (&w)[NB], const uint32_t (&high)[2][4], const uint32_t (&zero)[4],
                                          float2 (&acc)[NB][16], int gr, int c) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint2 v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = 8 * (i >> 1) + 2 * c + (i & 1);
      v[i] = *reinterpret_cast<const uint2*>(stage + key * 128 + ((gr ^ (2 * c + (i & 1))) << 4) + 8 * (half ^ (gr >> 1 & 1)));
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      uint32_t t[4][4];
#pragma unroll
      for (int z = 0; z < 4; ++z)
        y == 0 ? transpose_bytes(v[4 * z].x, v[4 * z + 1].x, v[4 * z + 2].x, v[4 * z + 3].x, t[z])
               : transpose_bytes(v[4 * z].y, v[4 * z + 1].y, v[4 * z + 2].y, v[4 * z + 3].y, t[z]);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        int lm[NB][4], hi[4];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
#pragma unroll
          for (int b = 0; b < NB; ++b) mma_i8<false>(lm[b], z == 0, zero, w[b].p[z], t[2 * z][x], t[2 * z + 1][x]);
          mma_i8<false>(hi, z == 0, zero, high[z], t[2 * z][x], t[2 * z + 1][x]);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const float2 z = k8_join(lm[b][0], lm[b][1], lm[b][2], lm[b][3], hi[2 * b], hi[2 * b + 1]);
          float2& o = acc[b][8 * half + 4 * y + x];
          o = sm100::ffma2(o, make_float2(w[b].before, w[b].before), sm100::fmul2(z, make_float2(w[b].now, w[b].now)));
        }
      }
    }
  }
}

// Few rows: up to 8 NB of them in an item, whose keys are dealt out to four warps with rings of their own.  With `cut` the quanta of all tiles,
// one after the other, are dealt out in equal shares, and a CTA takes a share for one group of heads, so that none has more to do than another
// whatever the lengths; an item that goes over the end of a share goes on in the next, and attn_kv8_join_kernel adds its pieces up.  Without, an
// item a CTA.  The heads of a share are neighbours among the CTAs: they read the same rows at the same time, 128 bytes each (with shares of
// all items, heads one after the other, memory delivered 555 MB for 423, and 24 sequences of up to 4096 keys with 32 heads took 140 us).
template <typename T, int NB>
__global__ void __launch_bounds__(kK8Threads, K8Ring<NB>::kCtas)
attn_kv8_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Kv8Attn a) {
  extern __shared__ __align__(1024) uint8_t sm[];
  constexpr int kStages = K8Ring<NB>::kStages, R = 8 * NB, LD = kK8SlotRow;
  K8Ring<NB>& ring = *reinterpret_cast<K8Ring<NB>*>(sm + K8Ring<NB>::kBytes);
  if (threadIdx.x == 0) {
    for (int w = 0; w < 4; ++w)
      for (int i = 0; i < kStages; ++i) sm100::mbar_init(&ring.full[w][i], 1);
    sm100::fence_barrier_init();
    sm100::tma_prefetch_desc(&tmK);
    sm100::tma_prefetch_desc(&tmV);
    ring.gave_up = 0;
  }
  __syncthreads();
  chain_enter();
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, gr = lane >> 2, c = lane & 3;
  const int n_x = a.cu != nullptr ? a.n_seq * a.tiles : a.n, hs = k8_groups(a.H, a.c.G), rep = a.H / a.c.G, groups = hs / a.c.G;
  if (a.cu != nullptr) {                               // rows behind the last sequence, by all CTAs (by one, 4096 of 32 heads took 550 us)
    T* out = reinterpret_cast<T*>(a.out);
    const long long per = (long long)a.H * a.c.dv, first = (long long)blockIdx.x * kK8Threads + threadIdx.x;
    for (long long i = min(max(a.cu[a.n_seq], 0), a.n) * per + first; i < a.n * per; i += (long long)gridDim.x * kK8Threads) out[i] = from_f<T>(0.f);
  }
  const int hg = blockIdx.x % hs, share = blockIdx.x / hs, g = hg / groups, h0 = g * rep + hg % groups * kK8Heads;
  const int nh = min(kK8Heads, (g + 1) * rep - h0);
  int x = share, q0 = 0, left = 0x7fffffff, all = 0, shares = 1;
  if (a.cut) {
    // where the share begins: a lane counts the quanta of its tiles, and walks them if it is there; every warp for itself, without a barrier
    const int chunk = (n_x + 31) / 32, first = min(lane * chunk, n_x), last = min(first + chunk, n_x);
    int mine = 0;
    for (int i = first; i < last; ++i) mine += K8Tile(a, i).cost();
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += y;
    }
    all = __shfl_sync(0xffffffffu, before, 31);
    before -= mine;
    shares = max(1, min((int)gridDim.x / hs, all));    // none is empty
    const int begin = k8_share(share, all, shares);
    left = share < shares ? k8_share(share + 1, all, shares) - begin : 0;
    if (threadIdx.x == 0) reinterpret_cast<K8Cut*>(a.part + (size_t)gridDim.x * 2 * R * LD)[blockIdx.x].more = 0;
    if (left <= 0) return;
    const bool here = begin >= before && begin < before + mine;
    x = first;
    q0 = begin - before;
    if (here) {
      for (; x < last - 1; ++x) {
        const int q = K8Tile(a, x).cost();
        if (q0 < q) break;
        q0 -= q;
      }
    }
    const int who = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    if (who < 0) return;
    x = __shfl_sync(0xffffffffu, x, who);
    q0 = __shfl_sync(0xffffffffu, q0, who);
  }
  uint8_t* stages = sm + warp * kK8Stage * kStages;
  volatile int* gave_up = &ring.gave_up;
  // Copies run ahead of the arithmetic by up to a ring, into the next piece too, but for one stage, which the sums of a piece go through.
  int taken = 0, sent = 0;                             // stages waited for, and stages that copies were sent to
  int s_row, s_left, n_row = 0, n_units = 0;           // the copies' next row, and stages left in their piece; the next piece's
  auto send = [&](int ahead) {                         // until `ahead` stages are on their way
    while (sent - taken < ahead) {
      if (s_left == 0) {
        if (n_units == 0) return;
        s_row = n_row;
        s_left = 2 * n_units;
        n_units = 0;
      }
      if (lane == 0) {                                 // rows past the range are whatever lies there: they are not seen
        uint64_t* bar = &ring.full[warp][sent % kStages];
        sm100::mbar_expect_tx(bar, kK8Stage);
        sm100::tma_load_3d(stages + sent % kStages * kK8Stage, s_left & 1 ? &tmV : &tmK, bar, 0, g, s_row);
      }
      if (s_left & 1) s_row += kK8Quantum;
      --s_left;
      ++sent;
    }
  };
  uint32_t none[4], zero[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    zero[i] = k8_kept(kMagic);
    none[i] = k8_kept(0);
  }
  bool failed = false, fresh = true;
  while (true) {
    const K8Piece p(a, x, q0, left);
    if (p.q1 == p.q0) return;                          // an item without rows (the shares have none), or a share that ends where an item begins
    if (threadIdx.x == 0) {
      ring.piece[0] = p.t.r0;
      ring.piece[1] = (p.t.r1 - p.t.r0) * nh;
      ring.piece[2] = p.q0;
      ring.piece[3] = p.behind;
    }
    const int mine = p.units(warp), k0 = p.k0() + warp * kK8Keys, k1 = p.k1(), rows = (p.t.r1 - p.t.r0) * nh;
    if (fresh) {
      s_row = p.t.base + k0;
      s_left = 2 * mine;
      fresh = false;
    }
    left -= p.t.cost() - p.behind - q0;
    send(kStages);
    // queries, scales and the next piece: what they need comes from memory together
    K8Query<T> query[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int m = min(b * 8 + gr, rows - 1);         // rows past the end repeat the last
      query[b].load(a, p.t.r0 + m / nh, h0 + m % nh, c);
    }
    float kn[2], vn[2];                                // scales of keys `lane` and lane + 32 of the next unit
    auto load_scales = [&](int i) {
      if (i < mine) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const size_t at = (size_t)((p.t.base + min(k0 + i * kK8Quantum + 32 * y + lane, k1 - 1)) >> a.c.shift) * a.c.G + g;
          kn[y] = a.c.ks[at];
          vn[y] = a.c.vs[at];
        }
      }
    };
    load_scales(0);
    const int x1 = left > 0 && a.cut ? k8_next(a, n_x, x) : n_x;
    const bool more = x1 < n_x;
    if (more) {                                        // the next piece, for the copies
      const K8Piece n(a, x1, 0, left);
      n_units = n.units(warp);
      n_row = n.t.base + n.k0() + warp * kK8Keys;
    }
    K8Rows r[NB];
    float2 acc[NB][16];
    uint32_t q_high[4][4];                             // high bytes of the first group, and of the second or nothing
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      k8_rows<T>(a, query[b], r[b]);
#pragma unroll
      for (int y = 0; y < 16; ++y) acc[b][y] = make_float2(0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int y = 0; y < 4; ++y) q_high[i][y] = y & 1 ? (NB == 2 ? r[NB - 1].high[i][y >> 1] : k8_kept(0)) : r[0].high[i][y >> 1];
    const int seen_by_all = min(p.t.len0, k1), seen_from = max(0, p.t.len1 - a.window);
    for (int i = 0; i < mine; ++i) {
      float s[NB][16];
      const float km[2] = {kn[0], kn[1]}, vm[2] = {vn[0], vn[1]};
      load_scales(i + 1);
      const int key0 = k0 + i * kK8Quantum, ahead = i < mine - 1 ? kStages : kStages - 1;
      failed = !sm100::mbar_wait_warp(&ring.full[warp][taken % kStages], (taken / kStages) & 1, gave_up);
      if (failed) break;
      k8_scores<NB>(stages + taken % kStages * kK8Stage, r, q_high, zero, s, gr, c);
      sm100::fence_proxy_async_smem();                 // these reads before the copy that goes over them
      __syncwarp();
      ++taken;
      send(ahead);
      K8Weights w[NB];
      float ks[16], vs[16];
      k8_scales(km, a.c.shift, c, ks);
      k8_scales(vm, a.c.shift, c, vs);
#pragma unroll
      for (int b = 0; b < NB; ++b) k8_softmax(a, r[b], s[b], ks, vs, key0, c, key0 + kK8Keys > seen_by_all || key0 < seen_from, w[b]);
      failed = !sm100::mbar_wait_warp(&ring.full[warp][taken % kStages], (taken / kStages) & 1, gave_up);
      if (failed) break;
      uint32_t high[2][4];
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        const int z = y >> 2, half = y >> 1 & 1;
        high[z][y & 3] = !(y & 1) ? w[0].high[z][half] : NB == 2 ? w[NB - 1].high[z][half] : none[y >> 1];
      }
      k8_values<NB>(stages + taken % kStages * kK8Stage, w, high, zero, acc, gr, c);
      sm100::fence_proxy_async_smem();
      __syncwarp();
      ++taken;
      send(ahead);
    }
    if (failed) *gave_up = 1;
    // the warps' shares, in the stage that no copy is on its way to
    const int idle = (taken + kStages - 1) % kStages;
    if (lane == 0) ring.free_stage[warp] = idle;
    auto sums_of = [&](int w, int stage) { return reinterpret_cast<float*>(sm + (w * kStages + stage) * kK8Stage); };
    auto stats_of = [&](int w, int stage) {
      return K8Ring<NB>::kStatHere ? ring.stat + w * R : reinterpret_cast<float2*>(sm + (w * kStages + stage) * kK8Stage + K8Ring<NB>::kSumBytes);
    };
    float* sums = sums_of(warp, idle);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      r[b].l += __shfl_xor_sync(0xffffffffu, r[b].l, 1);
      r[b].l += __shfl_xor_sync(0xffffffffu, r[b].l, 2);
      const int m = b * 8 + gr;
      if (c == 0) stats_of(warp, idle)[m] = make_float2(r[b].m, r[b].l);
#pragma unroll
      for (int y = 0; y < 16; y += 4) {
        const int i = 8 * c + 2 * ((y >> 3) ^ (c & 1)) + (y >> 2 & 1);
        *reinterpret_cast<float4*>(sums + k8_sum_at(m, i)) = make_float4(acc[b][y].x, acc[b][y + 1].x, acc[b][y + 2].x, acc[b][y + 3].x);
        *reinterpret_cast<float4*>(sums + k8_sum_at(m, i + 4)) = make_float4(acc[b][y].y, acc[b][y + 1].y, acc[b][y + 2].y, acc[b][y + 3].y);
      }
    }
    __syncthreads();
    if (*gave_up) break;
    const int r0 = ring.piece[0], n_rows = ring.piece[1], began = ring.piece[2], behind = ring.piece[3];
    const bool whole = began == 0 && behind == 0;
    float* slot = whole ? nullptr : a.part + ((size_t)blockIdx.x * 2 + (began == 0)) * R * LD;
    if (!whole && began == 0 && threadIdx.x == 0) {    // its last quantum is the share's of which the first is not behind it
      const long long last = k8_share(share + 1, all, shares) + behind - 1ll;
      const int more_shares = (int)(((last + 1) * shares - 1) / all) - share;
      reinterpret_cast<K8Cut*>(a.part + (size_t)gridDim.x * 2 * R * LD)[blockIdx.x] = K8Cut{r0, n_rows, h0, nh, more_shares};
    }
    const float* from[4];
    const float2* stats[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int stage = ring.free_stage[y];
      from[y] = sums_of(y, stage);
      stats[y] = stats_of(y, stage);
    }
    for (int m = warp; m < n_rows; m += 4) {
      float w[4], mx = -INFINITY, l = 0.f;
#pragma unroll
      for (int y = 0; y < 4; ++y) mx = fmaxf(mx, stats[y][m].x);
      const int h = h0 + m % nh;
      const float sk = whole && a.sink != nullptr ? a.sink[h] * kLog2e : -INFINITY, top = fmaxf(mx, sk), ref = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        w[y] = exp2f(stats[y][m].x - ref);
        l = fmaf(stats[y][m].y, w[y], l);
      }
      const float den = whole ? l + exp2f(sk - ref) : 1.f, f = den == 0.f ? 0.f : 1.f / den;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float4 v = *reinterpret_cast<const float4*>(from[y] + k8_sum_at(m, lane));
        o = make_float4(fmaf(v.x, w[y], o.x), fmaf(v.y, w[y], o.y), fmaf(v.z, w[y], o.z), fmaf(v.w, w[y], o.w));
      }
      if (whole) {
        k8_store_row<T>(a, r0 + m / nh, h, lane, make_float4(o.x * f, o.y * f, o.z * f, o.w * f));
      } else {
        *reinterpret_cast<float4*>(slot + m * LD + 4 * lane) = o;
        if (lane == 0) {
          slot[m * LD + kK8Dim] = mx;
          slot[m * LD + kK8Dim + 1] = l;
        }
      }
    }
    if (!more) return;
    sm100::fence_proxy_async_smem();                   // these reads before copies
    __syncthreads();
    x = x1;
    q0 = 0;
  }
  // a copy did not arrive: those in flight land before the CTA ends
  if (threadIdx.x == 0) {
    atomicCAS(a.err, 0, kK8Wait);
    const unsigned long long t0 = sm100::globaltimer_ns();
    while (sm100::globaltimer_ns() - t0 < 200000ull) {
    }
  }
  __syncthreads();
}

// Joins the pieces of the items that shares cut.  A CTA the item that begins in the share (and heads) of its number, if that one was cut.
// A row has W warps, each with every W-th piece, eight of which are under way together: one long sequence has some fifty.  The CTAs are
// small enough to be resident all at once, most of them have nothing to do (as CTAs of 1024 threads, in three rounds, they took 12 us).
constexpr int kK8JoinThreads = 512;
template <typename T, int R>
__global__ void __launch_bounds__(kK8JoinThreads, 2) attn_kv8_join_kernel(const __grid_constant__ Kv8Attn a) {
  chain_enter();
  constexpr int W = kK8JoinThreads / 32 / R;
  __shared__ float4 sums[W][R][32];
  __shared__ float2 stat[W][R];
  const int hs = k8_groups(a.H, a.c.G);
  const K8Cut cut = reinterpret_cast<const K8Cut*>(a.part + (size_t)gridDim.x * 2 * R * kK8SlotRow)[blockIdx.x];
  const int m = (threadIdx.x >> 5) % R, mine = (threadIdx.x >> 5) / R, lane = threadIdx.x & 31;
  if (cut.more == 0) return;
  const int pieces = cut.more + 1, h = cut.h0 + m % cut.nh;
  const float* const slots = a.part + m * kK8SlotRow;
  if (m < cut.rows) {
    const float sk = mine == 0 && a.sink != nullptr ? a.sink[h] * kLog2e : -INFINITY;
    float top = sk, l = sk == -INFINITY ? 0.f : 1.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = mine; i0 < pieces; i0 += W * 8) {
      float4 v[8];
      float2 st[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = min(i0 + W * i, pieces - 1);
        const float* s = slots + ((size_t)(blockIdx.x + at * hs) * 2 + (at == 0)) * R * kK8SlotRow;
        v[i] = *reinterpret_cast<const float4*>(s + 4 * lane);
        st[i] = *reinterpret_cast<const float2*>(s + kK8Dim);
      }
      float now = top;
#pragma unroll
      for (int i = 0; i < 8; ++i) now = fmaxf(now, st[i].x);
      const float ref = now == -INFINITY ? 0.f : now, al = exp2f(top - ref);
      top = now;
      l *= al;
      o = make_float4(o.x * al, o.y * al, o.z * al, o.w * al);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i0 + W * i < pieces) {
          const float e = exp2f(st[i].x - ref);
          l = fmaf(st[i].y, e, l);
          o = make_float4(fmaf(v[i].x, e, o.x), fmaf(v[i].y, e, o.y), fmaf(v[i].z, e, o.z), fmaf(v[i].w, e, o.w));
        }
      }
    }
    sums[mine][m][lane] = o;
    if (lane == 0) stat[mine][m] = make_float2(top, l);
  }
  __syncthreads();
  if (m >= cut.rows || mine != 0) return;
  float top = stat[0][m].x, den = 0.f;
#pragma unroll
  for (int y = 1; y < W; ++y) top = fmaxf(top, stat[y][m].x);
  const float ref = top == -INFINITY ? 0.f : top;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int y = 0; y < W; ++y) {
    const float4 v = sums[y][m][lane];
    const float e = exp2f(stat[y][m].x - ref);
    o = make_float4(fmaf(v.x, e, o.x), fmaf(v.y, e, o.y), fmaf(v.z, e, o.z), fmaf(v.w, e, o.w));
    den = fmaf(stat[y][m].y, e, den);
  }
  const float f = den == 0.f ? 0.f : 1.f / den;
  k8_store_row<T>(a, cut.r0 + m / cut.nh, h, lane, make_float4(o.x * f, o.y * f, o.z * f, o.w * f));
}

// How a call runs: tokens of a tile, tiles of a sequence, groups of 8 rows, CTAs, and whether their shares cut items.
struct K8Plan {
  int tt, tiles, nb, ctas, cut;
};
static K8Plan k8_plan(int n, int n_seq, int max_q, int H, int G, int max_len, int window) {
  K8Plan p{};
  const int nh = std::min(H / G, kK8Heads);
  const bool one = n_seq <= 0 || max_q <= 1;
  p.tt = one ? 1 : std::max(1, std::min(max_q, 16 / nh));
  p.tiles = one ? 1 : (max_q + p.tt - 1) / p.tt;
  p.nb = p.tt * nh <= 8 ? 1 : 2;
  if (window > 0) max_len = std::min<long long>(max_len, (long long)window + p.tt + kK8Keys);      // rows see windows that start apart
  const long long x = n_seq > 0 ? (long long)n_seq * p.tiles : n, hs = k8_groups(H, G), quanta = std::max(1, (max_len + kK8Quantum - 1) / kK8Quantum),
                  resident = (long long)kNumSMs * (p.nb == 1 ? K8Ring<1>::kCtas : K8Ring<2>::kCtas);
  if (x * hs > 0x7fffffff || x * (quanta + 2) > 0x7fffffff) return p;      // not to be counted in 32 bits: ctas 0
  // Up to 1024 keys an item a CTA: the join is a launch, 4 us.  Us cut | not (sequences of so many keys, 32 heads on 8): 1 of 500 9.4 | 7.2, of 1000
  // 10.7 | 10.6, of 1500 11.0 | 13.9; 16 of 500 12.3 | 8.3, of 1000 13.2 | 12.7, of 1500 13.6 | 16.7; 64 of 700 22.4 | 19.1, of 1000 25.4 | 23.9, of
  // 2000 36 | 40; 64 of 1000, 32 on 32, 72 | 70, of 2000 107 | 108.
  p.cut = quanta > 4;
  p.ctas = (int)std::min<long long>((p.cut ? std::min(std::max(1ll, resident / hs), x * quanta) : x) * hs, 0x7fffffff);
  return p;
}
static size_t k8_part_floats(const K8Plan& p) { return p.cut ? (size_t)p.ctas * (2 * 8 * p.nb * kK8SlotRow + sizeof(K8Cut) / 4) : 0; }

int make_tmap_bytes_heads(CUtensorMap* map, const void* ptr, uint64_t dim, uint64_t heads, uint64_t rows, uint32_t box_rows);

template <typename T, int NB>
static int launch_attn_kv8(const Kv8Attn& a, const K8Plan& p, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t stream) {
  static SmemLimit limit;
  if (const int e = allow_smem(attn_kv8_kernel<T, NB>, k8_smem<NB>(), limit)) return e;
  launch_chained(attn_kv8_kernel<T, NB>, p.ctas, kK8Threads, k8_smem<NB>(), stream, tk, tv, a);
  if (p.cut) launch_chained(attn_kv8_join_kernel<T, 8 * NB>, p.ctas, kK8JoinThreads, 0, stream, a);
  return launch_status();
}

}  // namespace ell

using namespace ell;

// The arguments come as structures of 64-bit words: from Python thirty words of one object cost less than thirty arguments.
struct Kv8Args {                  // a cache: rows, scales, heads and head sizes, rows that share a scale, rows in all
  int8_t *k, *v;
  float *ks, *vs;
  long long G, d, dv, block, rows;
};
struct Kv8AppendCall {
  Kv8Args c;
  const void *k, *v;
  const int *base, *len, *cu;
  long long n, n_seq, max_new, ldk, ldv, is_bf16;
  int* err;
};
struct Kv8ReadCall {
  Kv8Args c;
  void *k, *v;
  const int *base, *len, *cu;
  int* row_base;
  long long n, rows_q, max_len, is_bf16;
  int* err;
};
struct Kv8AttnCall {
  Kv8Args c;
  const void* q;
  void* out;
  float* part;
  long long part_floats;
  const int *base, *len;
  const float *sink, *slopes;
  const int* cu;
  long long n, n_seq, max_q, H, ldq, max_len, window, is_bf16;
  int* err;
  double scale;
};
static_assert(sizeof(Kv8Args) == 9 * 8 && sizeof(Kv8AppendCall) == 21 * 8 && sizeof(Kv8ReadCall) == 20 * 8 && sizeof(Kv8AttnCall) == 28 * 8, "");
static bool k8_cache(const Kv8Args& a, Kv8Cache& c) {
  const bool ok = a.G > 0 && a.G <= 65535 && a.d > 0 && a.dv > 0 && a.d <= kK8Dim && a.dv <= kK8Dim && a.block > 0 && a.block <= kK8MaxBlock &&
                  !(a.block & (a.block - 1)) && a.rows % a.block == 0 && a.rows <= 0x7fffffff && aligned_to(a.k, 16) && aligned_to(a.v, 16);
  int shift = 0;
  while ((1ll << shift) < a.block) ++shift;
  c = Kv8Cache{a.k, a.v, a.ks, a.vs, a.rows, (int)a.G, (int)a.d, (int)a.dv, shift};
  return ok;
}

// The rows k [n, G, d], v [n, G, dv] (rows of ldk / ldv elements) of a step: those of cu[i] .. cu[i + 1] - 1 go to the places
// len[cu[i]] - 1 and on of the sequence whose rows start at base[cu[i]].  max_new bounds their number.
ELL_API int ell_kv8_append(const Kv8AppendCall* call, cudaStream_t stream) {
  const Kv8AppendCall& x = *call;
  Kv8Cache c;
  if (x.n <= 0 || x.n_seq <= 0) return 0;
  if (!k8_cache(x.c, c) || x.n > 0x7fffffff) return -2;
  const int esz = x.is_bf16 ? 2 : 4;
  // a bound below 1 is that of sequences without rows: one that has some all the same is found out by the first block's CTAs
  const long long blocks = (std::max(x.max_new, 1ll) + 2 * x.c.block - 2) / x.c.block, ctas = blocks * ((2 * c.G + 7) / 8);
  if (ctas > 0x7fffffff || x.n_seq > 65535) return -2;
  const bool vec = c.d % 8 == 0 && c.dv % 8 == 0 && x.ldk * esz % 16 == 0 && x.ldv * esz % 16 == 0 && aligned_to(x.k, 16) && aligned_to(x.v, 16);
#define ELL_APPEND(T, V)                                                                                                                \
  launch_chained(kv8_append_kernel<T, V>, dim3((unsigned)ctas, (unsigned)x.n_seq), 256, 0, stream, c, (const T*)x.k, (const T*)x.v,      \
                 x.base, x.len, x.cu, (int)x.n, (int)blocks, (int)x.ldk, (int)x.ldv, x.err)
  if (x.is_bf16) vec ? ELL_APPEND(__nv_bfloat16, 8) : ELL_APPEND(__nv_bfloat16, 1);
  else vec ? ELL_APPEND(float, 8) : ELL_APPEND(float, 1);
#undef ELL_APPEND
  return launch_status();
}

// cu [n + 1] and row_base [2, rows_q] (or null, null): see kv8_read_kernel.
ELL_API int ell_kv8_read(const Kv8ReadCall* call, cudaStream_t stream) {
  const Kv8ReadCall& x = *call;
  Kv8Cache c;
  if (x.n <= 0 || x.max_len <= 0) return 0;
  if (!k8_cache(x.c, c) || x.n > 65535 || x.max_len > 0x3fffffff || (x.cu != nullptr && x.n * x.max_len > 0x7fffffff)) return -2;
  const int vec = c.d % 8 == 0 && c.dv % 8 == 0 ? 8 : 1;
  // a thread takes eight positions (the prefixes beside kv8_read_kernel took 31 us so, 32 with sixteen, 35 with thirty-two)
  const int per = c.G * (c.d + c.dv) / vec, beside = std::max(1, 256 / per), z = (beside * per + 255) / 256, chunk = 8 * beside;
  if (z > 65535) return -2;
  const dim3 grid((unsigned)((x.max_len + chunk - 1) / chunk), (unsigned)x.n, (unsigned)z);
#define ELL_READ(T, V)                                                                                                                  \
  launch_chained(kv8_read_kernel<T, V>, grid, 256, 0, stream, c, (T*)x.k, (T*)x.v, x.base, x.len, x.cu, x.row_base, (int)x.rows_q,      \
                 (int)x.max_len, chunk, x.err)
  if (x.is_bf16) vec == 8 ? ELL_READ(__nv_bfloat16, 8) : ELL_READ(__nv_bfloat16, 1);
  else vec == 8 ? ELL_READ(float, 8) : ELL_READ(float, 1);
#undef ELL_READ
  return launch_status();
}

// out bf16 [n, width]
ELL_API int ell_kv8_clear(void* out, const int* len, const int* cu, int n_seq, int n, int width, cudaStream_t stream) {
  if (n <= 0) return 0;
  launch_chained(kv8_clear_kernel, grid_for((long long)n * 32, 256, 4), 256, 0, stream, (__nv_bfloat16*)out, len, cu, n_seq, n, width);
  return launch_status();
}

// q rows of ldq elements.  max_len bounds len[].  part (16-byte aligned): `part_floats` of scratch where max_len is above 1024, enough for
// max(296, key heads x groups of 16 query heads) x 4232.  window: keys a row sees (<= 0: all).  cu [n_seq + 1] (or null): rows
// cu[i] .. cu[i + 1] - 1 are consecutive tokens of one sequence, with one base and lengths that grow by one; max_q bounds their number.
// There is one sequence at least where there are borders.
ELL_API int ell_attn_kv8(const Kv8AttnCall* call, cudaStream_t stream) {
  const Kv8AttnCall& x = *call;
  Kv8Attn a{};
  if (x.n <= 0) return 0;
  if (!k8_cache(x.c, a.c) || x.n > 0x7fffffff || x.H <= 0 || x.H > 0x7fffff || x.H % x.c.G) return -2;
  if (x.max_len > 0x3fffffff || x.max_q > 0x3fffffff) return -2;
  if (x.cu != nullptr && (x.n_seq <= 0 || x.n_seq > 0x7fffffff)) return -2;      // borders without a sequence: a tile would look behind them
  const int n_seq = x.cu == nullptr ? 0 : (int)x.n_seq;
  const K8Plan p = k8_plan((int)x.n, n_seq, (int)x.max_q, (int)x.H, a.c.G, (int)x.max_len, (int)std::min(x.window, 0x3fffffffll));
  if (p.ctas <= 0) return -2;
  if (p.cut && (x.part == nullptr || !aligned_to(x.part, 16) || (size_t)x.part_floats < k8_part_floats(p))) return -2;
  a.q = x.q, a.out = x.out, a.part = x.part, a.base = x.base, a.len = x.len, a.cu = x.cu, a.sink = x.sink, a.slopes = x.slopes;
  a.n = (int)x.n, a.H = (int)x.H, a.ldq = (int)x.ldq, a.n_seq = n_seq, a.tiles = p.tiles, a.tt = p.tt, a.cut = p.cut;
  a.max_len = (int)std::max(x.max_len, 0ll);
  a.window = x.window > 0 ? (int)std::min(x.window, 0x3fffffffll) : 0x3fffffff;
  a.scale = (float)(x.scale * 1.4426950408889634 / 2097152);
  a.err = x.err;
  CUtensorMap tk, tv;
  int rc = make_tmap_bytes_heads(&tk, a.c.k, k8_row(a.c.d), a.c.G, a.c.rows, kK8Keys);
  if (!rc) rc = make_tmap_bytes_heads(&tv, a.c.v, k8_row(a.c.dv), a.c.G, a.c.rows, kK8Keys);
  if (rc) return rc;
  if (x.is_bf16) return p.nb == 1 ? launch_attn_kv8<__nv_bfloat16, 1>(a, p, tk, tv, stream) : launch_attn_kv8<__nv_bfloat16, 2>(a, p, tk, tv, stream);
  return p.nb == 1 ? launch_attn_kv8<float, 1>(a, p, tk, tv, stream) : launch_attn_kv8<float, 2>(a, p, tk, tv, stream);
}
