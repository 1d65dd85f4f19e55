// Rows of a matrix in the registers of a few lanes: loads and stores of rows of any width on any element boundary, sums
// over the lanes that hold a row, a workgroup's parameter sums.  Used by the row norms (norm.hip, rms.hip).
#pragma once
#include <type_traits>

#include "common.h"
#include "../../include/e2v2.h"

namespace e2v2 {

// out_a[c] = the sum over the n_part rows of part [a][n_part][w] for a < arrays (1 or 2), in order, rounded once to the
// output's type; NULL outputs are left out (norm.hip)
int launch_param_sums(const float* part, int n_part, int w, int arrays, void* out0, int type0, void* out1, int type1,
                      hipStream_t s);

namespace {

inline int type_size(int t) { return t == E2V2_F32 ? 4 : 2; }
inline bool type_ok(int t) { return t == E2V2_F32 || t == E2V2_BF16 || t == E2V2_F16; }

template <typename T>
struct RowVec {
  static constexpr int n = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
  typedef T any __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));   // on any element boundary
  typedef float ftype __attribute__((ext_vector_type(16 / sizeof(T))));
};

// The lane's columns: vector k starts at column (l + k kL) V.
template <int V, int kL, int NV, typename F>
__device__ __forceinline__ void each_vec(int l, F&& f) {
#pragma unroll
  for (int k = 0; k < NV; ++k) f(k, (l + k * kL) * V);
}

// The same with whole = true_type for a vector that every lane has in full, false_type where elements from w on have to
// be left out: masks on every element made 6,007 x 5001 bf16 rows bound by the VALU.
template <int V, int kL, int NV, typename F>
__device__ __forceinline__ void each_vec(int l, int w, F&& f) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (l + k * kL) * V;
    if ((k + 1) * kL * V <= w) f(k, c, std::true_type{});
    else f(k, c, std::false_type{});
  }
}

// A lane's vectors of a row of w >= V elements (any w for V = 1).  All loads are unconditional, so that those of a
// row's operands are in flight together: a vector that would pass the end starts V before it instead (a branch would
// wait for its load in place: 100,000 x 129 fp32 backward 57 us).  get() then moves what belongs to the row down and,
// with kClear, clears the rest.
template <typename T, int V, int kL, int NV>
struct RowLoad {
  typename RowVec<T>::type raw[V > 1 ? NV : 1];
  T one[V > 1 ? 1 : NV];

  __device__ __forceinline__ void load(const T* row, int l, int w) {
    each_vec<V, kL, NV>(l, [&](int k, int c) {
      if constexpr (V > 1) raw[k] = *reinterpret_cast<const typename RowVec<T>::any*>(row + min(c, w - V));
      else one[k] = row[min(c, w - 1)];
    });
  }

  template <bool kClear = true>
  __device__ __forceinline__ void get(int l, int w, float (&out)[NV * V]) const {
    each_vec<V, kL, NV>(l, [&](int k, int c) {
      if constexpr (V > 1) {
        const auto f = __builtin_convertvector(raw[k], typename RowVec<T>::ftype);
#pragma unroll
        for (int e = 0; e < V; ++e) out[k * V + e] = f[e];
      } else {
        out[k] = (float)one[k];
      }
    });
    const int past = w % V ? V - w % V : 0;        // elements by which the row's last vector starts early
    each_vec<V, kL, NV>(l, w, [&](int k, int c, auto whole) {
      if constexpr (decltype(whole)::value) return;
      float* v = out + k * V;
      const bool moved = c < w && c + V > w;
#pragma unroll
      for (int d = V / 2; d > 0; d /= 2) {
        if (past & d) {
#pragma unroll
          for (int e = 0; e < V; ++e) v[e] = moved ? (e + d < V ? v[e + d] : 0.f) : v[e];
        }
      }
      if constexpr (kClear) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = c < w ? v[e] : 0.f;
      }
    });
  }
};

// The lane's V elements from column c on, or those of them that the row has: pieces of a half, a quarter, ... of a
// vector as the bits of w % V say.
template <typename T, int V>
__device__ __forceinline__ void store_row(const float* v, T* row, int c, int w, bool whole) {
  if constexpr (V == 1) {
    if (c < w) row[c] = (T)v[0];
  } else {
    T o[V];
#pragma unroll
    for (int k = 0; k < V; ++k) o[k] = (T)v[k];
    if (whole || c + V <= w) {
      typename RowVec<T>::type f;
#pragma unroll
      for (int k = 0; k < V; ++k) f[k] = o[k];
      *reinterpret_cast<typename RowVec<T>::any*>(row + c) = f;
    } else if (c < w) {
      T* at = row + c;
      auto piece = [&](auto size) {
        constexpr int D = decltype(size)::value;
        if constexpr (D < V) {
          if (w & D) {
            typedef T part __attribute__((ext_vector_type(D), aligned(sizeof(T))));
            part f;
#pragma unroll
            for (int k = 0; k < D; ++k) f[k] = o[k];
            *reinterpret_cast<part*>(at) = f;
            at += D;
#pragma unroll
            for (int k = 0; k + D < V; ++k) o[k] = o[k + D];
          }
        }
      };
      piece(std::integral_constant<int, 4>{});
      piece(std::integral_constant<int, 2>{});
      piece(std::integral_constant<int, 1>{});
    }
  }
}

// v + its partner's, kLanes lanes away, by an exchange of rows of 16 lanes or of halves in registers (no trip through
// LDS).  The results are taken as integers first: a bit cast of a vector's element casts element 0 here.
template <int kLanes>
__device__ __forceinline__ float swap_sum(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  uint32_t lo, hi;
  if constexpr (kLanes == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    lo = r[0], hi = r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    lo = r[0], hi = r[1];
  }
  return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}

// a b, rounded by itself: fused with the subtraction of its own row mean it would leave the rounding where the
// difference is zero.
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// Sums of K values over the kL lanes that hold a row, in every lane.  red: two buffers of [K][waves], used in turn, so
// that one barrier a sum is enough (a buffer is written again two sums later, behind the barrier between).
template <int kL, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float (*red)[4][16], int& turn) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if constexpr (kL >= 2) v[k] += dpp_mov<0xB1>(v[k]);    // lane ^ 1
    if constexpr (kL >= 4) v[k] += dpp_mov<0x4E>(v[k]);    // lane ^ 2
    if constexpr (kL >= 8) v[k] += dpp_mov<0x141>(v[k]);   // the other half of 8
    if constexpr (kL >= 16) v[k] += dpp_mov<0x140>(v[k]);  // the other half of 16
    if constexpr (kL >= 32) v[k] = swap_sum<16>(v[k]);
    if constexpr (kL >= 64) v[k] = swap_sum<32>(v[k]);
  }
  if constexpr (kL > 64) {
    constexpr int kWaves = kL / 64;
    const int wv = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) red[turn][k][wv] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) v[k] += red[turn][k][i];
    }
    turn ^= 1;
  }
}

template <typename W, int V, int kL, int NV>
__device__ __forceinline__ void load_params_as(const W* p, int l, int w, float (&out)[NV * V]) {
  typedef W any __attribute__((ext_vector_type(V), aligned(sizeof(W))));
  each_vec<V, kL, NV>(l, [&](int k, int c) {
    if (c + V <= w) {
      const any v = *reinterpret_cast<const any*>(p + c);
#pragma unroll
      for (int e = 0; e < V; ++e) out[k * V + e] = (float)v[e];
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) out[k * V + e] = c + e < w ? (float)p[c + e] : 0.f;
    }
  });
}

// The lane's elements of a parameter vector (NULL: the value of an absent one).
template <int V, int kL, int NV>
__device__ __forceinline__ void load_params(const void* p, int type, int l, int w, float absent, float (&out)[NV * V]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < NV * V; ++e) out[e] = absent;
  } else if (type == E2V2_F32) {
    load_params_as<float, V, kL, NV>(static_cast<const float*>(p), l, w, out);
  } else if (type == E2V2_BF16) {
    load_params_as<__bf16, V, kL, NV>(static_cast<const __bf16*>(p), l, w, out);
  } else {
    load_params_as<_Float16, V, kL, NV>(static_cast<const _Float16*>(p), l, w, out);
  }
}

// Adds the workgroup's row groups' parameter sums (those of a wavefront in registers, then the four wavefronts') and
// writes them as partial row blockIdx.x.
template <int V, int kL, int NV>
__device__ __forceinline__ void write_part(const float (&acc)[NV * V], int l, int w, float* out) {
  if constexpr (kL > 64) {
    each_vec<V, kL, NV>(l, [&](int k, int c) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (c + e < w) out[c + e] = acc[k * V + e];
    });
  } else {
    constexpr int kC = kL * NV * V;
    __shared__ float red[4][kC];
    const int wv = threadIdx.x >> 6;
    const bool mine = (threadIdx.x & 63) < kL;
    __syncthreads();
    each_vec<V, kL, NV>(l, [&](int k, int c) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float v = acc[k * V + e];
        if constexpr (kL <= 2) v += dpp_mov<0x4E>(v);      // lane ^ 2
        if constexpr (kL <= 4) v += dpp_mov<0x124>(v);     // four lanes round a row of 16
        if constexpr (kL <= 8) v += dpp_mov<0x128>(v);     // eight lanes round
        if constexpr (kL <= 16) v = swap_sum<16>(v);
        if constexpr (kL <= 32) v = swap_sum<32>(v);
        if (mine) red[wv][c + e] = v;
      }
    });
    __syncthreads();
    for (int c = threadIdx.x; c < w; c += 256) out[c] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
  }
}

// Lanes that hold a row, and 16-byte vectors a lane holds of it.  Up to 1024 elements a part of a wavefront, so that
// no barrier stands in the way: of the shapes that hold the row one with few idle places (400,000 x 129 bf16 forward:
// 52 us on 8 lanes of 3 vectors, 82 on 32 of one; 100,000 x 129 fp32: 24 on 16 of 3, 41 on 64 of one).  Wider rows
// take a workgroup of 256, up to 32 elements a lane (6,007 x 5001 bf16 forward: 35 us, on 1024 lanes 45; second order,
// 4,000 x 8192 fp32: 147 and 188), in the backward pass with its two sums a column 16 (fp32: 6,007 x 5001 85 us with
// 24, 79 on 1024 lanes) or 24 (bf16: 4,000 x 8192 64 us with 32, 56 on 1024 lanes).
struct RowShape {
  int lanes, vecs;       // vecs 0: rows shorter than a vector, one element a lane
};

inline RowShape row_shape(int w, int v, bool bwd) {
  if (w < v) return {w <= 2 ? 2 : w <= 4 ? 4 : 8, 0};
  const int nv = (w + v - 1) / v;
  if (nv <= 8) return {nv <= 2 ? 2 : nv <= 4 ? 4 : 8, 1};
  if (nv <= 12) return {4, 3};
  if (nv <= 16) return {16, 1};
  if (nv <= 24) return {8, 3};
  if (nv <= 32) return {32, 1};
  if (nv <= 48) return {16, 3};
  if (nv <= 64) return {64, 1};
  if (nv <= 96) return {32, 3};
  if (nv <= 128) return {64, 2};
  if (w <= 1024) return {64, nv <= 192 ? 3 : 4};
  if (w <= (!bwd ? 8192 : v == 8 ? 6144 : 4096)) {
    for (int k = 1;; k = k < 4 ? k + 1 : 8)
      if (nv <= 256 * k) return {256, k};
  }
  return {1024, w <= 8192 ? 8 / v : 16 / v};
}

}  // namespace
}  // namespace e2v2
