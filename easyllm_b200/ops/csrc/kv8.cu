// A key/value cache held in 8 bits: written, read back, attended over.
//
// Rows k [R, G, dk], v [R, G, dv] of int8 (dk, dv: the head sizes rounded up to 16), and a scale for each block of `block` rows
// and head, [R / block, G], fp32.  A scale is a power of two s = 2^e, e >= -126, the least with max|x| <= 127 s (at most 2^121, where
// q is cut to 127: 128 2^121 is past the end of fp32 and bf16); x = q s, |q| <= 127.
// So x / s and q s_old / s are exact but for one rounding to an integer, and q s is exact in bf16 and in fp32: reading back loses
// nothing, and a block that rows join later is off by less than s (s / 2 + s / 4 + ..: a scale that grows at least doubles).
// A block that got a value that is not finite has the scale NaN and reads as NaN.
#include <algorithm>

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
  const int lane = threadIdx.x & 31, g = (int)(item % c.G), block = 1 << c.shift;
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
struct Kv8Attn {
  Kv8Cache c;
  const void* q;
  void* out;                      // [n, H, dv]
  float* part;
  const int *base, *len, *cu;
  const float *sink, *slopes;
  int n, H, ldq, n_seq, splits, range, window;
  float scale;
  int* err;
};

// A warp a query row and head, key by key.
template <typename T>
__global__ void __launch_bounds__(128) attn_kv8_kernel(const Kv8Attn a) {
  chain_enter();
  const long long item = blockIdx.x * 4ll + (threadIdx.x >> 5);
  if (item >= (long long)a.n * a.H) return;
  const int t = (int)(item / a.H), h = (int)(item % a.H), lane = threadIdx.x & 31, g = h / (a.H / a.c.G);
  int len = a.cu != nullptr && t >= a.cu[a.n_seq] ? 0 : a.len[t];
  const int base = a.base[t];
  if (len > 0 && !k8_inside(a.c, base, len)) {
    if (lane == 0) atomicCAS(a.err, 0, kK8Place);
    len = 0;
  }
  const int dk = k8_row(a.c.d), dv = k8_row(a.c.dv);
  float q[4], acc[4], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int x = lane + 32 * i;
    q[i] = x < a.c.d ? to_f<T>(reinterpret_cast<const T*>(a.q)[(size_t)t * a.ldq + (size_t)h * a.c.d + x]) : 0.f;
    acc[i] = 0.f;
  }
  for (int p = max(0, len - a.window); p < len; ++p) {
    const size_t row = (size_t)base + p;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 32 * i < a.c.d) s = fmaf(q[i], (float)a.c.k[(row * a.c.G + g) * dk + lane + 32 * i], s);
    s = warp_sum(s) * a.c.ks[(row >> a.c.shift) * a.c.G + g] * a.scale;
    if (a.slopes != nullptr) s += a.slopes[h] * (float)(p - (len - 1));
    const float now = fmaxf(m, s), al = m == now ? 1.f : expf(m - now), w = expf(s - now), f = w * a.c.vs[(row >> a.c.shift) * a.c.G + g];
    m = now;
    l = l * al + w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 32 * i < a.c.dv) acc[i] = fmaf(f, (float)a.c.v[(row * a.c.G + g) * dv + lane + 32 * i], acc[i] * al);
  }
  float f = l == 0.f ? 0.f : 1.f / l;
  if (a.sink != nullptr && l != 0.f) {
    const float sk = a.sink[h], mm = fmaxf(m, sk);
    f = expf(m - mm) / (l * expf(m - mm) + expf(sk - mm));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < a.c.dv) reinterpret_cast<T*>(a.out)[((size_t)t * a.H + h) * a.c.dv + lane + 32 * i] = from_f<T>(l == 0.f ? 0.f : acc[i] * f);
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

ELL_API int ell_attn_kv8(const void* q, const int8_t* kc, const int8_t* vc, const float* ks, const float* vs, void* out, const int* base,
                         const int* len, const float* sink, const float* slopes, const int* cu, int n, int n_seq, int max_q, int H, int G, int d, int dv,
                         int ldq, int max_len, int window, float scale, int shift, long long rows, int is_bf16, int* err, cudaStream_t stream) {
  if (n <= 0) return 0;
  if (!k8_sizes_ok(G, d, dv, shift) || H % G) return -2;
  Kv8Attn a{};
  a.c = Kv8Cache{const_cast<int8_t*>(kc), const_cast<int8_t*>(vc), const_cast<float*>(ks), const_cast<float*>(vs), rows, G, d, dv, shift};
  a.q = q, a.out = out, a.base = base, a.len = len, a.cu = cu, a.sink = sink, a.slopes = slopes;
  a.n = n, a.H = H, a.ldq = ldq, a.n_seq = n_seq, a.window = window > 0 ? window : 0x7fffffff, a.scale = scale, a.err = err;
  const unsigned ctas = (unsigned)(((long long)n * H + 3) / 4);
  if (is_bf16) launch_chained(attn_kv8_kernel<__nv_bfloat16>, ctas, 128, 0, stream, a);
  else launch_chained(attn_kv8_kernel<float>, ctas, 128, 0, stream, a);
  return launch_status();
}
