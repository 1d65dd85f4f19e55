// Root-mean-square norm of rows [n][w] in fp32, bf16 or fp16 with the residual's addition before it, its output in the
// rows' type or in 8 bits with scales, and its backward pass.  With <.> the mean over a row:
//   forward   h = x + res (rounded to the rows' type, as the next layer reads it; the norm is of that h),
//             r = (<h^2> + eps)^(-1/2),  y = h r w
//   backward  u = gy w,  gx = r (u - h r <u h r>) + gh  (the gradient of x and of res),  gw = sum_rows gy h r
// Statistics and sums are fp32; y, gx and gw are rounded once.  The 8-bit output is taken from y in fp32, so it too is
// rounded once (quant8.h has the format).
//
// One pass over memory, as in the layer norm (rows.h): a row stays in the registers of 2 to 1024 lanes.  A block of 128
// columns is 16 or 32 neighbouring lanes (or part of a lane's vectors), so a block's largest value takes DPP steps
// and no memory.  Bound: HBM.  With the residual, 32768 x 2048 bf16 forward 90 us (6.0 TB/s), backward 115 (4.7) and the
// weight's sums 5; 16384 x 4096 bf16 with 8-bit output 98 (4.8; on the same tensors again and again 67, from the cache).
#include <algorithm>

#include "quant8.h"
#include "rows.h"

namespace e2v2 {
namespace {

constexpr int kRmsMaxWidth = 16384;
constexpr int kRmsMaxParts = 1024;     // workgroups of a backward pass that leaves weight sums, at most (rms_grid)

struct RmsArgs {
  const void* x; const void* res; const void* w;
  void* h; void* y; uint8_t* scales; float* rstd;
  const void* gy; const void* gh; void* gx; float* part;
  int64_t n, ldx, ldres, ldgy, ldgh, ldy;
  int width, w_type;
  float eps;
};

// The largest bits of each vector's block of 128 columns, from those of the vectors themselves.
template <int V, int kL, int NV>
__device__ __forceinline__ void block_max(uint32_t (&m)[NV]) {
  constexpr int G = kBlock8 / V;                   // lanes of a block
#pragma unroll
  for (int k = 0; k < NV; ++k) m[k] = lanes_max<(kL < G ? kL : G)>(m[k]);
  if constexpr (kL < G && NV > 1) {                // a block spans several of a lane's vectors
    uint32_t a[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      a[k] = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (k * kL * V / kBlock8 == j * kL * V / kBlock8) a[k] = max(a[k], m[j]);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) m[k] = a[k];
  }
}

// A row's codes and scale bytes (row `at` of a table of n rows, the rows' bytes of a block side by side): whole vectors,
// into the row's padding too (rows of codes lie a multiple of 16 bytes apart).  What the padding holds is left open: codes
// of zero times the row's factor as far as vectors reach, and in rows of up to 8 columns old bytes; readers mask it.
template <int V, int kL, int NV>
__device__ __forceinline__ void store_codes(const float (&y)[NV * V], int l, int w, uint8_t* row, int64_t ld,
                                            uint8_t* scales, int64_t at, int64_t n) {
  uint32_t m[NV];
  auto largest = [&](auto bits) {
    uint32_t all = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      m[k] = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) m[k] = max(m[k], bits(y[k * V + e]));
      all = max(all, m[k]);
    }
    return all;
  };
  top_bits(largest);
  block_max<V, kL, NV>(m);
  each_vec<V, kL, NV>(l, [&](int k, int c) {
    const int s = scale_byte(m[k]);
    const float up = scale_up(s);
    if constexpr (V == 1) {
      if (c < w) row[c] = (uint8_t)codes4(y[k] * up, 0.f, 0.f, 0.f);
    } else if (c < ld) {
      uint32_t q[V / 4];
#pragma unroll
      for (int e = 0; e < V; e += 4)
        q[e / 4] = codes4(y[k * V + e] * up, y[k * V + e + 1] * up, y[k * V + e + 2] * up, y[k * V + e + 3] * up);
      if constexpr (V == 4) *reinterpret_cast<uint32_t*>(row + c) = q[0];
      else *reinterpret_cast<uint2*>(row + c) = make_uint2(q[0], q[1]);
    }
    if (c % kBlock8 == 0 && c < w) scales[c / kBlock8 * n + at] = (uint8_t)s;
  });
}

template <typename T, int V, int kL, int NV, bool kRes, bool kOut8>
__global__ __launch_bounds__(kL > 64 ? kL : 256) void k_rms_fwd(RmsArgs P) {
  constexpr int kR = kL > 64 ? 1 : 256 / kL, E = NV * V;
  __shared__ float red[2][4][16];
  const int l = threadIdx.x % kL, rg = threadIdx.x / kL, w = P.width;
  float g[E];
  load_params<V, kL, NV>(P.w, P.w_type, l, w, 1.f, g);
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kR + rg; row < P.n; row += (int64_t)gridDim.x * kR) {
    float h[E], s[1] = {0.f};
    RowLoad<T, V, kL, NV> rx, rr;
    rx.load(static_cast<const T*>(P.x) + row * P.ldx, l, w);
    if constexpr (kRes) rr.load(static_cast<const T*>(P.res) + row * P.ldres, l, w);
    rx.get(l, w, h);
    if constexpr (kRes) {
      float b[E];
      rr.get(l, w, b);
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] = (float)(T)(h[e] + b[e]);
      T* hr = static_cast<T*>(P.h) + row * w;
      each_vec<V, kL, NV>(l, w, [&](int k, int c, auto whole) { store_row<T, V>(h + k * V, hr, c, w, whole); });
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s[0] = fmaf(h[e], h[e], s[0]);
    group_sum<kL, 1>(s, red, turn);
    const float r = 1.0f / sqrtf(s[0] / (float)w + P.eps);
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] = h[e] * r * g[e];
    if constexpr (kOut8) {
      store_codes<V, kL, NV>(h, l, w, static_cast<uint8_t*>(P.y) + row * P.ldy, P.ldy, P.scales, row, P.n);
    } else {
      T* yr = static_cast<T*>(P.y) + row * w;
      each_vec<V, kL, NV>(l, w, [&](int k, int c, auto whole) { store_row<T, V>(h + k * V, yr, c, w, whole); });
      if (P.rstd && l == 0) P.rstd[row] = r;
    }
  }
}

template <typename T, int V, int kL, int NV, bool kGh>
__global__ __launch_bounds__(kL > 64 ? kL : 256) void k_rms_bwd(RmsArgs P) {
  constexpr int kR = kL > 64 ? 1 : 256 / kL, E = NV * V;
  __shared__ float red[2][4][16];
  const int l = threadIdx.x % kL, rg = threadIdx.x / kL, w = P.width;
  float g[E], ag[E];
  load_params<V, kL, NV>(P.w, P.w_type, l, w, 1.f, g);
#pragma unroll
  for (int e = 0; e < E; ++e) ag[e] = 0.f;
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kR + rg; row < P.n; row += (int64_t)gridDim.x * kR) {
    const float r = P.rstd[row];
    float hh[E], u[E], s[1] = {0.f};
    RowLoad<T, V, kL, NV> rh, ry, rg_;
    rh.load(static_cast<const T*>(P.x) + row * P.ldx, l, w);
    ry.load(static_cast<const T*>(P.gy) + row * P.ldgy, l, w);
    if constexpr (kGh) rg_.load(static_cast<const T*>(P.gh) + row * P.ldgh, l, w);
    rh.template get<false>(l, w, hh);              // past the row's end gy is zero, and so is all that h enters
    ry.get(l, w, u);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      hh[e] *= r;
      ag[e] = fmaf(u[e], hh[e], ag[e]);
      u[e] *= g[e];
      s[0] = fmaf(u[e], hh[e], s[0]);
    }
    group_sum<kL, 1>(s, red, turn);
    const float m = s[0] / (float)w;
#pragma unroll
    for (int e = 0; e < E; ++e) u[e] = r * (u[e] - hh[e] * m);
    if constexpr (kGh) {
      float b[E];
      rg_.template get<false>(l, w, b);
#pragma unroll
      for (int e = 0; e < E; ++e) u[e] += b[e];
    }
    T* o = static_cast<T*>(P.gx) + row * w;
    each_vec<V, kL, NV>(l, w, [&](int k, int c, auto whole) { store_row<T, V>(u + k * V, o, c, w, whole); });
  }
  if (P.part) write_part<V, kL, NV>(ag, l, w, P.part + (int64_t)blockIdx.x * w);
}

enum class RmsPass { kFwd, kFwd8, kBwd };

template <RmsPass kPass, typename T, int V, int kL, int NV>
void rms_launch(const RmsArgs& P, unsigned grid, hipStream_t s) {
  const dim3 block(kL > 64 ? kL : 256);
  if constexpr (kPass == RmsPass::kBwd) {
    if (P.gh) hipLaunchKernelGGL((k_rms_bwd<T, V, kL, NV, true>), dim3(grid), block, 0, s, P);
    else hipLaunchKernelGGL((k_rms_bwd<T, V, kL, NV, false>), dim3(grid), block, 0, s, P);
  } else {
    constexpr bool k8 = kPass == RmsPass::kFwd8;
    if (P.res) hipLaunchKernelGGL((k_rms_fwd<T, V, kL, NV, true, k8>), dim3(grid), block, 0, s, P);
    else hipLaunchKernelGGL((k_rms_fwd<T, V, kL, NV, false, k8>), dim3(grid), block, 0, s, P);
  }
}

template <RmsPass kPass, typename T>
void rms_dispatch(const RmsArgs& P, unsigned grid, hipStream_t s) {
  constexpr int V = RowVec<T>::n;
  constexpr bool kBwd = kPass == RmsPass::kBwd;
  const RowShape f = row_shape(P.width, V, kBwd);
  switch (f.lanes * 16 + f.vecs) {
    case 2 * 16: return rms_launch<kPass, T, 1, 2, 1>(P, grid, s);
    case 4 * 16: return rms_launch<kPass, T, 1, 4, 1>(P, grid, s);
    case 8 * 16: return rms_launch<kPass, T, 1, 8, 1>(P, grid, s);
    case 2 * 16 + 1: return rms_launch<kPass, T, V, 2, 1>(P, grid, s);
    case 4 * 16 + 1: return rms_launch<kPass, T, V, 4, 1>(P, grid, s);
    case 8 * 16 + 1: return rms_launch<kPass, T, V, 8, 1>(P, grid, s);
    case 16 * 16 + 1: return rms_launch<kPass, T, V, 16, 1>(P, grid, s);
    case 32 * 16 + 1: return rms_launch<kPass, T, V, 32, 1>(P, grid, s);
    case 4 * 16 + 3: return rms_launch<kPass, T, V, 4, 3>(P, grid, s);
    case 8 * 16 + 3: return rms_launch<kPass, T, V, 8, 3>(P, grid, s);
    case 16 * 16 + 3: return rms_launch<kPass, T, V, 16, 3>(P, grid, s);
    case 64 * 16 + 1: return rms_launch<kPass, T, V, 64, 1>(P, grid, s);
    case 32 * 16 + 3: return rms_launch<kPass, T, V, 32, 3>(P, grid, s);
    case 64 * 16 + 2: return rms_launch<kPass, T, V, 64, 2>(P, grid, s);
  }
  if constexpr (V == 4) {
    switch (f.lanes * 16 + f.vecs) {
      case 64 * 16 + 3: return rms_launch<kPass, T, V, 64, 3>(P, grid, s);
      case 64 * 16 + 4: return rms_launch<kPass, T, V, 64, 4>(P, grid, s);
      case 256 * 16 + 8:
        if constexpr (!kBwd) return rms_launch<kPass, T, V, 256, 8>(P, grid, s);
    }
  }
  switch (f.lanes * 16 + f.vecs) {
    case 256 * 16 + 1:
      if constexpr (V == 8) return rms_launch<kPass, T, V, 256, 1>(P, grid, s);
      break;
    case 256 * 16 + 2: return rms_launch<kPass, T, V, 256, 2>(P, grid, s);
    case 256 * 16 + 3: return rms_launch<kPass, T, V, 256, 3>(P, grid, s);
    case 256 * 16 + 4:
      if constexpr (!kBwd || V == 4) return rms_launch<kPass, T, V, 256, 4>(P, grid, s);
      break;
    case 1024 * 16 + 8 / V:
      if constexpr (kBwd) return rms_launch<kPass, T, V, 1024, 8 / V>(P, grid, s);
      break;
    default: return rms_launch<kPass, T, V, 1024, 16 / V>(P, grid, s);
  }
}

template <RmsPass kPass>
void rms_run(const RmsArgs& P, int type, unsigned grid, hipStream_t s) {
  if (type == E2V2_F32) rms_dispatch<kPass, float>(P, grid, s);
  else if (type == E2V2_BF16) rms_dispatch<kPass, __bf16>(P, grid, s);
  else rms_dispatch<kPass, _Float16>(P, grid, s);
}

// Workgroups of a pass: they stride over the rows with the weight loaded once, as in the layer norm.
unsigned rms_grid(int64_t n, int width, int type, bool bwd, bool sums) {
  const RowShape f = row_shape(width, 16 / type_size(type), bwd);
  const int r = f.lanes > 64 ? 1 : 256 / f.lanes;
  int64_t most = f.lanes == 1024 ? 512 : f.lanes == 256 ? 2048 : 1024;
  if (sums) most = f.lanes == 1024 ? 256 : f.vecs <= 1 ? 1024 : 512;
  else if (bwd && f.lanes <= 32 && f.vecs <= 1) most = 1 << 23;
  return (unsigned)std::min<int64_t>((n + r - 1) / r, most);
}

int rms_check(const char* what, const e2v2_rms_rows_args* a) {
  E2V2_REQUIRE(a, "%s: null arguments", what);
  E2V2_REQUIRE(a->n >= 0 && a->width > 0 && a->width <= kRmsMaxWidth, "%s: %lld rows of width %d (1 to %d)", what,
               (long long)a->n, a->width, kRmsMaxWidth);
  E2V2_REQUIRE(type_ok(a->type) && type_ok(a->w_type), "%s: types %d, %d", what, a->type, a->w_type);
  E2V2_REQUIRE(a->ldx >= 0 && a->ldres >= 0 && a->ldgy >= 0 && a->ldgh >= 0, "%s: negative row stride", what);
  const uintptr_t all = (uintptr_t)a->x | (uintptr_t)a->res | (uintptr_t)a->h | (uintptr_t)a->gy | (uintptr_t)a->gh |
                        (uintptr_t)a->gx | (a->scales ? 0 : (uintptr_t)a->y);
  E2V2_REQUIRE(all % type_size(a->type) == 0 && (uintptr_t)a->w % type_size(a->w_type) == 0 &&
                   (uintptr_t)a->rstd % 4 == 0, "%s: misaligned operand", what);
  return 0;
}

RmsArgs rms_args(const e2v2_rms_rows_args* a) {
  return RmsArgs{a->x, a->res, a->w, a->h, a->y, a->scales, a->rstd, a->gy, a->gh, a->gx, nullptr, a->n, a->ldx,
                 a->ldres, a->ldgy, a->ldgh, a->ldy, a->width, a->w_type, a->eps};
}

}  // namespace
}  // namespace e2v2

using namespace e2v2;

E2V2_API int e2v2_rms_rows_fwd(const e2v2_rms_rows_args* a, hipStream_t s) {
  if (const int rc = rms_check("rms_rows_fwd", a)) return rc;
  if (a->n == 0) return 0;
  E2V2_REQUIRE(a->x && a->y && (!a->res || a->h), "rms_rows_fwd: null operand");
  const RmsArgs P = rms_args(a);
  const unsigned grid = rms_grid(a->n, a->width, a->type, false, false);
  if (a->scales) {
    E2V2_REQUIRE(a->ldy >= a->width && a->ldy % 16 == 0 && (uintptr_t)a->y % 16 == 0,
                 "rms_rows_fwd: rows of codes lie a multiple of 16 bytes apart, got %lld", (long long)a->ldy);
    rms_run<RmsPass::kFwd8>(P, a->type, grid, s);
  } else {
    rms_run<RmsPass::kFwd>(P, a->type, grid, s);
  }
  E2V2_LAUNCHED("k_rms_fwd");
  return 0;
}

E2V2_API int64_t e2v2_rms_rows_workspace(int64_t n, int width) {
  if (n <= 0 || width <= 0) return 0;
  return std::min<int64_t>(n, kRmsMaxParts) * width * 4;
}

E2V2_API int e2v2_rms_rows_bwd(const e2v2_rms_rows_args* a, void* gw, float* ws, int64_t ws_bytes, hipStream_t s) {
  if (const int rc = rms_check("rms_rows_bwd", a)) return rc;
  E2V2_REQUIRE(a->n == 0 || (a->x && a->gy && a->gx && a->rstd), "rms_rows_bwd: null operand");
  E2V2_REQUIRE(!gw || (ws_bytes >= e2v2_rms_rows_workspace(a->n, a->width) && (ws || a->n == 0)),
               "rms_rows_bwd: workspace of %lld bytes", (long long)ws_bytes);
  RmsArgs P = rms_args(a);
  P.part = gw ? ws : nullptr;
  const unsigned grid = rms_grid(a->n, a->width, a->type, true, gw != nullptr);
  if (grid) {
    rms_run<RmsPass::kBwd>(P, a->type, grid, s);
    E2V2_LAUNCHED("k_rms_bwd");
  }
  return gw ? launch_param_sums(ws, (int)grid, a->width, 1, gw, a->w_type, nullptr, 0, s) : 0;
}
