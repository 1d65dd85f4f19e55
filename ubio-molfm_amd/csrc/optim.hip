// The parameter update of training over many tensors at once: the global norm of all gradients, their scaling by it,
// and AdamW steps with moments in 32 or in 8 bits.  With g the gradient, c = min(1, max_norm / (norm + 1e-6)) and step
// t:
//   m = b1 m + (1 - b1) c g,   v = b2 v + (1 - b2) (c g)^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
// Arithmetic is fp32 (the norm's sum fp64: it neither loses small tensors beside large ones nor overflows; 8-bit
// moments fp64 up to their code); bf16 and fp16 parameters are rounded to nearest once.  Every element is read and
// written once by one thread, the sums run in a fixed order: no atomics, results repeat bitwise.  Bound: HBM (241 M
// bf16 parameters with 32-bit moments 1.02 ms, 5.2 TB/s; 241 M fp32 parameters with 8-bit moments 0.76 ms, 5.1 TB/s;
// 24.5 M fp32 in 240 tensors 135 us, behind a norm, which leaves gradients in the caches, 124; the norm 18 to 32).
//
// The tensors are cut into chunks, one workgroup each.  What does not change from step to step (addresses and places
// of the parameters) is a table in device memory; the gradients' addresses, which may, come with the launch.  The step
// count is kept per chunk, so that each workgroup advances its own without waiting for another and a captured step
// counts its replays.
//
// Moments in 8 bits: runs of 32 consecutive elements share a scale byte s, 2^(s - 127) being the binade of the run's
// largest value; m has a sign, 4 exponent and 3 mantissa bits (code 0x80: NaN), v no sign, 5 exponent and 3 mantissa
// bits (code 255: NaN).  Moved by 2^(15 - s) or 2^(31 - s) a value's fp32 exponent field is the code's exponent field,
// subnormals included, so that encoding is one ldexp, an addition and a shift, and decoding the reverse.  The addition
// rounds stochastically: with b2 = 0.999 a step changes v by 0.1%, and rounding to the nearest of codes 6 to 12% apart
// would leave it where it is for ever; here the stored value's mean is the value.  A v above zero keeps a code above
// zero: zero would let the next step divide by eps.  The random bits are a hash of seed, step and element.  A value
// that is not finite becomes the NaN of its own element.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "common.h"
#include "../../include/e2v2.h"

namespace e2v2 {
namespace {

constexpr int kOptThreads = 256;
constexpr int kOptChunk = E2V2_OPT_CHUNK;
constexpr int kNormList = 256;         // gradients of a norm launch (a thread each finds the chunks' tensors)
constexpr int kNormChunk = 4096;
constexpr int kNormParts = 1024;       // workgroups of a norm launch at most
constexpr int kStepList = 384;         // gradients of a step launch (3 KB of the 4 KB of kernel arguments)

template <typename T>
struct Vec16 {
  static constexpr int n = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
  typedef T any __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));   // on any element boundary
  typedef float ftype __attribute__((ext_vector_type(16 / sizeof(T))));
};

// N elements at p, on any element boundary (the hardware takes 16 bytes unaligned).
template <typename T, int N>
__device__ __forceinline__ void load_n(const T* p, float (&out)[N]) {
  constexpr int V = Vec16<T>::n;
#pragma unroll
  for (int k = 0; k < N; k += V) {
    const typename Vec16<T>::type v = *reinterpret_cast<const typename Vec16<T>::any*>(p + k);
    const auto f = __builtin_convertvector(v, typename Vec16<T>::ftype);
#pragma unroll
    for (int e = 0; e < V; ++e) out[k + e] = f[e];
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_n(const float (&v)[N], T* p) {
  constexpr int V = Vec16<T>::n;
#pragma unroll
  for (int k = 0; k < N; k += V) {
    typename Vec16<T>::ftype f;
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = v[k + e];
    const typename Vec16<T>::type o = __builtin_convertvector(f, typename Vec16<T>::type);
    *reinterpret_cast<typename Vec16<T>::any*>(p + k) = o;
  }
}

// Elements i .. i + N of n at p, those past n zero; kWhole: all are there.
template <bool kWhole, typename T, int N>
__device__ __forceinline__ void load_some(const T* p, int i, int n, float (&out)[N]) {
  if (kWhole || i + N <= n) {
    load_n<T, N>(p + i, out);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = i + e < n ? (float)p[i + e] : 0.f;
  }
}

template <bool kWhole, typename T, int N>
__device__ __forceinline__ void store_some(const float (&v)[N], T* p, int i, int n) {
  if (kWhole || i + N <= n) {
    store_n<T, N>(v, p + i);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (i + e < n) p[i + e] = (T)v[e];
  }
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double red[kOptThreads / 64];
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < kOptThreads / 64; ++i) v += red[i];
  return v;
}

// The norm from its partial sums, in every thread.
__device__ __forceinline__ double norm_of_parts(const double* parts, int n) {
  double s = 0;
  for (int i = threadIdx.x; i < n; i += kOptThreads) s += parts[i];
  return sqrt(block_sum(s));
}

// The factor that brings a norm to max_norm (none: infinity), and a NaN for a NaN.
__device__ __forceinline__ double clip_factor(double norm, float max_norm) {
  const double c = (double)max_norm / (norm + 1e-6);
  return c < 1.0 || c != c ? c : 1.0;
}

// ---- norm and scaling of a list of tensors

struct NormArgs {
  void* p[kNormList];
  uint32_t numel[kNormList];
  int n;
  double* parts;                       // norm: written; scaling: read
  int n_parts;
  float max_norm;
  float* norm;
};

// Calls f(tensor, first element, elements) for every chunk of this workgroup.
template <typename F>
__device__ __forceinline__ void each_chunk(const NormArgs& P, F&& f) {
  __shared__ int first[kNormList + 1], wave_total[kNormList / 64];
  const int t = threadIdx.x;
  int c = t < P.n ? (int)((P.numel[t] + (uint32_t)kNormChunk - 1) / kNormChunk) : 0;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(c, o, 64);
    c += (t & 63) >= o ? up : 0;
  }
  if ((t & 63) == 63) wave_total[t >> 6] = c;
  __syncthreads();
  for (int w = 0; w < (t >> 6); ++w) c += wave_total[w];
  first[t + 1] = c;
  if (t == 0) first[0] = 0;
  __syncthreads();
  for (int chunk = blockIdx.x; chunk < first[kNormList]; chunk += gridDim.x) {
    int lo = 0, hi = kNormList;
    while (hi - lo > 1) {              // first[lo] <= chunk < first[hi]
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= chunk) lo = mid; else hi = mid;
    }
    const uint32_t at = (uint32_t)(chunk - first[lo]) * kNormChunk;
    f(lo, at, (int)min(P.numel[lo] - at, (uint32_t)kNormChunk));
  }
}

template <typename T>
__global__ __launch_bounds__(kOptThreads) void k_grad_norm(NormArgs P) {
  constexpr int N = 8;
  double s = 0;
  each_chunk(P, [&](int t, uint32_t at, int n) {
    const T* g = static_cast<const T*>(P.p[t]) + at;
    auto add = [&](auto whole) {
#pragma unroll
      for (int k = 0; k < kNormChunk / (kOptThreads * N); ++k) {
        const int i = (k * kOptThreads + threadIdx.x) * N;
        float v[N];
        load_some<decltype(whole)::value>(g, i, n, v);
#pragma unroll
        for (int e = 0; e < N; ++e) s = fma((double)v[e], (double)v[e], s);
      }
    };
    if (n == kNormChunk) add(std::true_type{});
    else add(std::false_type{});
  });
  s = block_sum(s);
  if (threadIdx.x == 0) P.parts[blockIdx.x] = s;
}

template <typename T>
__global__ __launch_bounds__(kOptThreads) void k_grad_scale(NormArgs P) {
  constexpr int N = 8;
  const double norm = norm_of_parts(P.parts, P.n_parts);
  const float c = (float)clip_factor(norm, P.max_norm);
  if (blockIdx.x == 0 && threadIdx.x == 0 && P.norm) *P.norm = (float)norm;
  each_chunk(P, [&](int t, uint32_t at, int n) {
    T* g = static_cast<T*>(P.p[t]) + at;
    auto scale = [&](auto whole) {
      constexpr int K = kNormChunk / (kOptThreads * N);
      float v[K][N];
#pragma unroll
      for (int k = 0; k < K; ++k) load_some<decltype(whole)::value>(g, (k * kOptThreads + threadIdx.x) * N, n, v[k]);
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[k][e] *= c;
        store_some<decltype(whole)::value>(v[k], g, (k * kOptThreads + threadIdx.x) * N, n);
      }
    };
    if (n == kNormChunk) scale(std::true_type{});
    else scale(std::false_type{});
  });
}

__global__ __launch_bounds__(kOptThreads) void k_norm_value(const double* parts, int n, float* norm) {
  const double v = norm_of_parts(parts, n);
  if (threadIdx.x == 0) *norm = (float)v;
}

// ---- codes of 8 bits

constexpr uint32_t kGolden = 0x9E3779B9u, kRoot2 = 0x6A09E667u, kRoot3 = 0xBB67AE85u;  // fractions of phi, 2^1/2, 3^1/2

__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x = (x ^ (x >> 16)) * kRoot2;
  x = (x ^ (x >> 15)) * kRoot3;
  return x ^ (x >> 16);
}

template <bool kSigned>
__device__ __forceinline__ float decode8(uint32_t code, int s) {
  const float t = __uint_as_float((kSigned ? code & 127u : code) << 20);
  const float x = ldexpf(t, s - (kSigned ? 15 : 31));
  if (code == (kSigned ? 128u : 255u)) return __uint_as_float(0x7FC00000u);
  return kSigned && code > 127u ? -x : x;
}

// u: 16 random bits.
template <bool kSigned>
__device__ __forceinline__ uint32_t encode8(float x, int s, uint32_t u) {
  const float t = ldexpf(fabsf(x), (kSigned ? 15 : 31) - s);
  uint32_t code = (__float_as_uint(t) + (u << 4) + 8u) >> 20;
  if (kSigned) code = code && x < 0.f ? code | 128u : code;
  else code = max(code, x > 0.f ? 1u : 0u);
  return fabsf(x) < __builtin_inff() ? code : (kSigned ? 128u : 255u);
}

// The scale byte of a run: its largest finite magnitude, over the four lanes that hold the run, stays below the last
// code of its binade or moves to the next.
template <bool kSigned>
__device__ __forceinline__ int scale8(const float (&x)[8]) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a = fabsf(x[e]);
    top = fmaxf(top, a < __builtin_inff() ? a : 0.f);
  }
  top = fmaxf(top, dpp_mov<0xB1>(top));
  top = fmaxf(top, dpp_mov<0x4E>(top));
  return (int)((__float_as_uint(top) + (kSigned ? 0x0FFFFFu : 0x1FFFFFu)) >> 23);
}

// ---- AdamW

struct StepArgs {
  const void* grad[kStepList];
  const e2v2_opt_chunk* chunks;
  int32_t* steps;
  void* m; void* v;
  uint8_t* ms; uint8_t* vs;
  const float* lr_dev;
  const double* parts;
  float* norm;
  int32_t* skipped;
  int n_parts, first_tensor, skip_nonfinite;
  uint32_t seed;
  float lr, b1, b2, one_b1, one_b2, ln_b1, ln_b2, eps, wd, max_norm;
  double b1d, b2d, one_b1d, one_b2d;
};

// a towards zero in fp32.
__device__ __forceinline__ float truncated(double a) {
  return (float)__builtin_bit_cast(double, __builtin_bit_cast(uint64_t, a) & ~0x1FFFFFFFull);
}

// The root of a >= 0.  The instruction takes numbers below the smallest normal one for zero; kTiny: they are moved up
// before (1 ulp, as the instruction).
template <bool kTiny>
__device__ __forceinline__ float root_of(float a) {
  if constexpr (!kTiny) return __builtin_amdgcn_sqrtf(a);
  const bool low = a < 0x1p-100f;
  const float r = __builtin_amdgcn_sqrtf(low ? a * 0x1p64f : a);
  return low ? r * 0x1p-32f : r;
}

struct StepFactors {
  double c;                            // of the gradients
  float size, root, decay;             // lr / (1 - b1^t), (1 - b2^t)^(-1/2), lr wd
  uint32_t key;
};

// One chunk.  kWhole: all of its elements are there; then the loads of both halves are in flight before the first is
// used.
template <bool kWhole, bool kTiny, typename T, int kBits>
__device__ __forceinline__ void adamw_chunk(const StepArgs& P, const StepFactors& F, const T* g, T* p, int n,
                                            int64_t off) {
  constexpr int N = 8, K = kOptChunk / (kOptThreads * N);
  float pv[K][N], gv[K][N], m[K][N], v[K][N];
  uint2 mc[K], vc[K];
  int ms[K], vs[K];
  // whole runs of 32, padded with zeros, take part: a run's lanes share its scale
  const int padded = kWhole ? kOptChunk : (n + 31) / 32 * 32;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = (k * kOptThreads + threadIdx.x) * N;
    if (!kWhole && i >= padded) break;
    load_some<kWhole>(p, i, n, pv[k]);
    load_some<kWhole>(g, i, n, gv[k]);
    if constexpr (kBits == 32) {
      load_n(static_cast<const float*>(P.m) + off + i, m[k]);
      load_n(static_cast<const float*>(P.v) + off + i, v[k]);
    } else {
      mc[k] = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(P.m) + off + i);
      vc[k] = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(P.v) + off + i);
      ms[k] = P.ms[(off + i) / 32];
      vs[k] = P.vs[(off + i) / 32];
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = (k * kOptThreads + threadIdx.x) * N;
    if (!kWhole && i >= padded) break;
    const int64_t at = off + i;
    if constexpr (kBits == 8) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        m[k][e] = decode8<true>((e < 4 ? mc[k].x : mc[k].y) >> (8 * (e % 4)) & 255u, ms[k]);
        v[k][e] = decode8<false>((e < 4 ? vc[k].x : vc[k].y) >> (8 * (e % 4)) & 255u, vs[k]);
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      float &a = m[k][e], &b = v[k][e];
      // the gap behind a tensor stays zero under a NaN factor too (masked at the moments' store instead: 241 M fp32 with
      // 8-bit moments 737 -> 751 us, by the other registers that whole chunks get)
      const bool there = kWhole || i + e < n;
      if constexpr (kBits == 32) {
        const float x = there ? gv[k][e] * (float)F.c : 0.f;
        a = fmaf(P.one_b1, x, P.b1 * a);
        b = fmaf(P.one_b2 * x, x, P.b2 * b);
      } else {
        // fp64 up to the code: truncated to fp32 a value keeps every bit that its code hangs on, so that the codes are
        // those of the exact moments (a value next to a border would take the other code by its fp32 rounding)
        const double x = there ? (double)gv[k][e] * F.c : 0.0;
        a = truncated(fma(P.one_b1d, x, P.b1d * (double)a));
        b = truncated(fma(P.one_b2d * x, x, P.b2d * (double)b));
      }
      pv[k][e] -= fmaf(F.decay, pv[k][e], F.size * (a * frcp(fmaf(root_of<kTiny>(b), F.root, P.eps))));
    }
    store_some<kWhole>(pv[k], p, i, n);
    if constexpr (kBits == 32) {
      store_n(m[k], static_cast<float*>(P.m) + at);
      store_n(v[k], static_cast<float*>(P.v) + at);
    } else {
      const int s = scale8<true>(m[k]), r = scale8<false>(v[k]);
      uint32_t mo[2] = {0, 0}, vo[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const uint32_t u = mix32((uint32_t)(at + e) ^ F.key);
        mo[e / 4] |= encode8<true>(m[k][e], s, u & 0xFFFFu) << (8 * (e % 4));
        vo[e / 4] |= encode8<false>(v[k][e], r, u >> 16) << (8 * (e % 4));
      }
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(P.m) + at) = make_uint2(mo[0], mo[1]);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(P.v) + at) = make_uint2(vo[0], vo[1]);
      if (i % 32 == 0) {
        P.ms[at / 32] = (uint8_t)s;
        P.vs[at / 32] = (uint8_t)r;
      }
    }
  }
}

template <typename T, int kBits, bool kTiny>
__global__ __launch_bounds__(kOptThreads) void k_adamw(StepArgs P) {
  const e2v2_opt_chunk ch = P.chunks[blockIdx.x];
  StepFactors F;
  F.c = 1.0;
  bool skip = false;
  if (P.parts) {
    const double norm = norm_of_parts(P.parts, P.n_parts);
    F.c = clip_factor(norm, P.max_norm);
    skip = P.skip_nonfinite && !(norm < (double)__builtin_inff());
    if (blockIdx.x == 0 && threadIdx.x == 0 && P.norm) {
      *P.norm = (float)norm;
      if (skip) *P.skipped += 1;
    }
  }
  const T* g = static_cast<const T*>(P.grad[ch.tensor - P.first_tensor]);
  if (skip || !g) return;
  const int t = P.steps[blockIdx.x] + 1;
  __syncthreads();
  if (threadIdx.x == 0) P.steps[blockIdx.x] = t;
  const float lr = P.lr_dev ? *P.lr_dev : P.lr;
  const float bc1 = -expm1f((float)t * P.ln_b1), bc2 = -expm1f((float)t * P.ln_b2);
  F.size = lr / bc1;
  F.root = 1.0f / sqrtf(bc2);
  F.decay = lr * P.wd;
  F.key = kBits == 8 ? mix32(mix32(P.seed) + (uint32_t)t * kGolden + (uint32_t)((uint64_t)ch.off >> 32) * kRoot2) : 0;
  T* p = static_cast<T*>(ch.p) + ch.at;
  if (ch.n == kOptChunk) adamw_chunk<true, kTiny, T, kBits>(P, F, g + ch.at, p, ch.n, ch.off);
  else adamw_chunk<false, kTiny, T, kBits>(P, F, g + ch.at, p, ch.n, ch.off);
}

// The values that codes stand for, eight a thread; exact in each of the three types as long as they are normal there.
template <typename T>
__global__ __launch_bounds__(kOptThreads) void k_moments(const uint8_t* mc, const uint8_t* ms, const uint8_t* vc,
                                                         const uint8_t* vs, T* m, T* v, int64_t n) {
  const int64_t i = ((int64_t)blockIdx.x * kOptThreads + threadIdx.x) * 8;
  if (i >= n) return;
  uint32_t c[2];
  float x[8];
  *reinterpret_cast<uint2*>(c) = *reinterpret_cast<const uint2*>(mc + i);
  int s = ms[i / 32];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = decode8<true>(c[e / 4] >> (8 * (e % 4)) & 255u, s);
  store_n<T, 8>(x, m + i);
  *reinterpret_cast<uint2*>(c) = *reinterpret_cast<const uint2*>(vc + i);
  s = vs[i / 32];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = decode8<false>(c[e / 4] >> (8 * (e % 4)) & 255u, s);
  store_n<T, 8>(x, v + i);
}

bool opt_type_ok(int t) { return t == E2V2_F32 || t == E2V2_BF16 || t == E2V2_F16; }

// Launches f(args, workgroups) for lists of at most kNormList tensors; those past 2^31 elements in pieces.
template <typename F>
int each_list(void* const* ptrs, const int64_t* numel, int n, int type, F&& f) {
  NormArgs P{};
  int64_t chunks = 0;
  const int size = type == E2V2_F32 ? 4 : 2;
  auto flush = [&]() -> int {
    if (!P.n) return 0;
    const int rc = f(P, (unsigned)std::min<int64_t>(chunks, kNormParts));
    P.n = 0;
    chunks = 0;
    return rc;
  };
  for (int t = 0; t < n; ++t) {
    if (!ptrs[t]) continue;
    for (int64_t at = 0; at < numel[t]; at += 1LL << 31) {
      P.p[P.n] = static_cast<char*>(ptrs[t]) + at * size;
      P.numel[P.n] = (uint32_t)std::min<int64_t>(numel[t] - at, 1LL << 31);
      chunks += (P.numel[P.n] + (int64_t)kNormChunk - 1) / kNormChunk;
      if (++P.n == kNormList)
        if (const int rc = flush()) return rc;
    }
  }
  return flush();
}

int list_check(const char* what, void* const* ptrs, const int64_t* numel, int n, int type) {
  E2V2_REQUIRE(n >= 0 && (n == 0 || (ptrs && numel)), "%s: %d tensors", what, n);
  E2V2_REQUIRE(opt_type_ok(type), "%s: type %d", what, type);
  for (int t = 0; t < n; ++t)
    E2V2_REQUIRE(numel[t] >= 0 && (uintptr_t)ptrs[t] % (type == E2V2_F32 ? 4 : 2) == 0,
                 "%s: tensor %d of %lld elements", what, t, (long long)numel[t]);
  return 0;
}

}  // namespace
}  // namespace e2v2

using namespace e2v2;

E2V2_API int e2v2_grad_norm_parts(const int64_t* numel, int n) {
  if (n <= 0 || !numel) return 0;
  int64_t entries = 0;
  for (int t = 0; t < n; ++t) entries += (numel[t] + (1LL << 31) - 1) >> 31;
  return (int)((entries + kNormList - 1) / kNormList * kNormParts);
}

E2V2_API int e2v2_grad_norm(void* const* grads, const int64_t* numel, int n, int type, double* parts, int capacity,
                            int* n_parts, hipStream_t s) {
  if (const int rc = list_check("grad_norm", grads, numel, n, type)) return rc;
  E2V2_REQUIRE(n_parts && *n_parts >= 0 && (parts || n == 0), "grad_norm: null operand");
  return each_list(grads, numel, n, type, [&](NormArgs& P, unsigned grid) -> int {
    E2V2_REQUIRE(*n_parts + (int)grid <= capacity, "grad_norm: room for %d partial sums", capacity);
    P.parts = parts + *n_parts;
    if (type == E2V2_F32) hipLaunchKernelGGL(k_grad_norm<float>, dim3(grid), dim3(kOptThreads), 0, s, P);
    else if (type == E2V2_BF16) hipLaunchKernelGGL(k_grad_norm<__bf16>, dim3(grid), dim3(kOptThreads), 0, s, P);
    else hipLaunchKernelGGL(k_grad_norm<_Float16>, dim3(grid), dim3(kOptThreads), 0, s, P);
    E2V2_LAUNCHED("k_grad_norm");
    *n_parts += (int)grid;
    return 0;
  });
}

E2V2_API int e2v2_grad_norm_value(const double* parts, int n_parts, float* norm, hipStream_t s) {
  E2V2_REQUIRE(n_parts >= 0 && (parts || n_parts == 0) && norm, "grad_norm_value: null operand");
  hipLaunchKernelGGL(k_norm_value, dim3(1), dim3(kOptThreads), 0, s, parts, n_parts, norm);
  E2V2_LAUNCHED("k_norm_value");
  return 0;
}

E2V2_API int e2v2_grad_scale(void* const* grads, const int64_t* numel, int n, int type, const double* parts,
                             int n_parts, float max_norm, float* norm, hipStream_t s) {
  if (const int rc = list_check("grad_scale", grads, numel, n, type)) return rc;
  E2V2_REQUIRE(n_parts >= 0 && (parts || n_parts == 0), "grad_scale: null operand");
  return each_list(grads, numel, n, type, [&](NormArgs& P, unsigned grid) -> int {
    P.parts = const_cast<double*>(parts);
    P.n_parts = n_parts;
    P.max_norm = max_norm;
    P.norm = norm;
    if (type == E2V2_F32) hipLaunchKernelGGL(k_grad_scale<float>, dim3(grid), dim3(kOptThreads), 0, s, P);
    else if (type == E2V2_BF16) hipLaunchKernelGGL(k_grad_scale<__bf16>, dim3(grid), dim3(kOptThreads), 0, s, P);
    else hipLaunchKernelGGL(k_grad_scale<_Float16>, dim3(grid), dim3(kOptThreads), 0, s, P);
    E2V2_LAUNCHED("k_grad_scale");
    return 0;
  });
}

E2V2_API int e2v2_adamw(const e2v2_adamw_args* a, hipStream_t s) {
  E2V2_REQUIRE(a, "adamw: null arguments");
  E2V2_REQUIRE(a->n_chunks >= 0 && a->n_chunks < 1 << 24 && a->n_tensors >= 0 && a->n_tensors <= kStepList,
               "adamw: %d chunks of %d tensors (at most %d)", a->n_chunks, a->n_tensors, kStepList);
  E2V2_REQUIRE(opt_type_ok(a->type) && (a->bits == 32 || a->bits == 8), "adamw: type %d, moments of %d bits", a->type,
               a->bits);
  if (a->n_chunks == 0) return 0;
  E2V2_REQUIRE(a->chunks && a->steps && a->grads && a->m && a->v && (a->bits == 32 || (a->ms && a->vs)),
               "adamw: null operand");
  E2V2_REQUIRE(((uintptr_t)a->m | (uintptr_t)a->v) % 16 == 0, "adamw: moments on 16-byte boundaries");
  E2V2_REQUIRE(a->n_parts >= 0 && (a->n_parts == 0 || a->parts) && (!a->skip_nonfinite || a->skipped),
               "adamw: null operand");
  E2V2_REQUIRE(a->beta1 >= 0 && a->beta1 < 1 && a->beta2 >= 0 && a->beta2 < 1, "adamw: betas %g, %g", a->beta1,
               a->beta2);
  StepArgs P{};
  const int size = a->type == E2V2_F32 ? 4 : 2;
  for (int t = 0; t < a->n_tensors; ++t) {
    E2V2_REQUIRE((uintptr_t)a->grads[t] % size == 0, "adamw: misaligned gradient %d", t);
    P.grad[t] = a->grads[t];
  }
  P.chunks = a->chunks;
  P.steps = a->steps;
  P.m = a->m; P.v = a->v; P.ms = a->ms; P.vs = a->vs;
  P.lr_dev = a->lr_dev;
  P.parts = a->n_parts ? a->parts : nullptr;
  P.norm = a->norm;
  P.skipped = a->skipped;
  P.n_parts = a->n_parts;
  P.first_tensor = a->first_tensor;
  P.skip_nonfinite = a->skip_nonfinite;
  P.seed = a->seed;
  P.lr = (float)a->lr;
  P.b1 = (float)a->beta1; P.b2 = (float)a->beta2;
  P.one_b1 = (float)(1 - a->beta1); P.one_b2 = (float)(1 - a->beta2);
  P.ln_b1 = (float)log(a->beta1); P.ln_b2 = (float)log(a->beta2);
  P.b1d = a->beta1; P.b2d = a->beta2;
  P.one_b1d = 1 - a->beta1; P.one_b2d = 1 - a->beta2;
  // frcp takes numbers below the smallest normal one for zero (roots are far above it)
  P.eps = a->eps > 0 ? std::max((float)a->eps, FLT_MIN) : 0.f;
  P.wd = (float)a->weight_decay;
  P.max_norm = a->max_norm;
  const dim3 grid(a->n_chunks), block(kOptThreads);
  auto go = [&](auto type, auto tiny) {
    using T = decltype(type);
    constexpr bool kTiny = decltype(tiny)::value;
    if (a->bits == 32) hipLaunchKernelGGL((k_adamw<T, 32, kTiny>), grid, block, 0, s, P);
    else hipLaunchKernelGGL((k_adamw<T, 8, kTiny>), grid, block, 0, s, P);
  };
  auto go_as = [&](auto tiny) {
    if (a->type == E2V2_F32) go(float{}, tiny);
    else if (a->type == E2V2_BF16) go(__bf16{}, tiny);
    else go(_Float16{}, tiny);
  };
  // Roots of v below 2^-126 are below 2^-63, and (1 - b2^t)^(-1/2) is largest in the first step: beside a larger eps they
  // round away.  With a smaller one, zero among them, the update would be too large or infinite.  (24.5 M parameters in
  // fp32: 125 us without, 128 with these roots or with a branch in the kernel.)
  if (a->eps < 0x1p-38 / sqrt(1 - a->beta2)) go_as(std::true_type{});
  else go_as(std::false_type{});
  E2V2_LAUNCHED("k_adamw");
  return 0;
}

E2V2_API int e2v2_moments(const uint8_t* mc, const uint8_t* ms, const uint8_t* vc, const uint8_t* vs, void* m, void* v,
                          int type, int64_t n, hipStream_t s) {
  E2V2_REQUIRE(n >= 0 && n % 32 == 0 && n < (1LL << 34) && opt_type_ok(type), "moments: %lld elements, type %d",
               (long long)n, type);
  if (n == 0) return 0;
  E2V2_REQUIRE(mc && ms && vc && vs && m && v, "moments: null operand");
  E2V2_REQUIRE(((uintptr_t)mc | (uintptr_t)vc) % 8 == 0 && ((uintptr_t)m | (uintptr_t)v) % 16 == 0,
               "moments: codes on 8-byte, values on 16-byte boundaries");
  const dim3 grid((unsigned)((n / 8 + kOptThreads - 1) / kOptThreads)), block(kOptThreads);
  if (type == E2V2_F32)
    hipLaunchKernelGGL(k_moments<float>, grid, block, 0, s, mc, ms, vc, vs, static_cast<float*>(m),
                       static_cast<float*>(v), n);
  else if (type == E2V2_BF16)
    hipLaunchKernelGGL(k_moments<__bf16>, grid, block, 0, s, mc, ms, vc, vs, static_cast<__bf16*>(m),
                       static_cast<__bf16*>(v), n);
  else
    hipLaunchKernelGGL(k_moments<_Float16>, grid, block, 0, s, mc, ms, vc, vs, static_cast<_Float16*>(m),
                       static_cast<_Float16*>(v), n);
  E2V2_LAUNCHED("k_moments");
  return 0;
}
