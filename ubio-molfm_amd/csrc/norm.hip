// Layer norm of rows [n][w] in fp32, bf16 or fp16, its backward pass with the weight's and the bias's gradients, and
// the derivative of that backward pass (force training differentiates the forces once more).  With <.> the mean over
// a row, xh = (x - <x>) r and r = (<(x - <x>)^2> + eps)^(-1/2):
//   forward        y = xh g + b
//   backward       u = gy g,  gx = r (u - <u> - xh <u xh>),  dg = sum_rows gy xh,  db = sum_rows gy
//   second order   (upstream qx, qg, qb of gx, dg, db)
//                  A = r (qx - <qx> - xh <qx xh>),  c = <u xh>,  m = <qx xh>,
//                  dgy = g A + qg xh + qb,  X = -r (c qx + m u) + qg gy,
//                  dx = r (X - <X> - xh <X xh>) - r <qx gx> xh,  d(g) = sum_rows gy A
// (<qx gx> is r (<qx u> - <qx> <u> - c m); d(b) is zero.)  Rows are rounded to their type once, at the store;
// statistics, row sums and the parameters' sums are fp32, the variance taken about the mean in a second pass over the
// registers (and the mean itself once more where a row is far narrower than it).
//
// One pass over memory: a row stays in the registers of kL lanes (2 to 64 of a wavefront, or a workgroup of 256 or
// 1024), read as 16-byte vectors on whatever element boundary the row starts (the hardware takes them unaligned); a
// row's last vector may start early, its end is stored in pieces.  A workgroup strides over the rows and keeps its
// columns' parameter sums in registers; each leaves one partial row, added in order by a second launch, so results
// repeat bitwise.  Bound: HBM (127,113 x 128 fp32: forward 24 us, 5.4 TB/s; backward 31 and its parameters' sums 4,
// 5.6; second order 53 and 4, 5.7; 32,768 x 2048 bf16: 47 us, 88 + 4 and 130 + 5, 5.7, 4.4 and 5.0 TB/s).
#include <algorithm>

#include "rows.h"

namespace e2v2 {
namespace {

constexpr int kLnMaxWidth = 16384;     // 1024 lanes of 16 elements
constexpr int kLnMaxParts = 1024;      // workgroups of a pass that leaves parameter sums, at most (ln_grid)

struct LnArgs {
  const void* x; const void* gy; const void* qx;
  const void* g; const void* b; const void* qg; const void* qb;
  void* y; void* gx;                 // forward: y; backward: gx; second order: y is dgy, gx is dx
  float* stats;                      // [n][2] mean, rstd
  float* part;                       // [2 or 1][gridDim.x][w], or NULL
  int64_t n, ldx, ldgy, ldq;
  int w, g_type, b_type;
  float eps;
};

template <typename T, int V, int kL, int NV>
__global__ __launch_bounds__(kL > 64 ? kL : 256) void k_layer_norm_fwd(LnArgs P) {
  constexpr int kR = kL > 64 ? 1 : 256 / kL, E = NV * V;
  __shared__ float red[2][4][16];
  const int l = threadIdx.x % kL, rg = threadIdx.x / kL, w = P.w;
  const float inv = 1.0f / (float)w;
  float g[E], b[E];
  load_params<V, kL, NV>(P.g, P.g_type, l, w, 1.f, g);
  load_params<V, kL, NV>(P.b, P.b_type, l, w, 0.f, b);
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kR + rg; row < P.n; row += (int64_t)gridDim.x * kR) {
    const T* xr = static_cast<const T*>(P.x) + row * P.ldx;
    float x[E], s[1] = {0.f}, q[1];
    RowLoad<T, V, kL, NV> rx;
    rx.load(xr, l, w);
    rx.get(l, w, x);
#pragma unroll
    for (int e = 0; e < E; ++e) s[0] += x[e];
    group_sum<kL, 1>(s, red, turn);
    float mean = s[0] / (float)w;             // a true quotient: exact for a row of one short value
    auto centre = [&](float by) {
      q[0] = 0.f;
      each_vec<V, kL, NV>(l, w, [&](int k, int c, auto whole) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          x[k * V + e] = whole || c + e < w ? x[k * V + e] - by : 0.f;
          q[0] = fmaf(x[k * V + e], x[k * V + e], q[0]);
        }
      });
      group_sum<kL, 1>(q, red, turn);
    };
    centre(mean);
    // Rows far narrower than their mean: what the sum's rounding left in it is taken off too.  It counts beside their
    // spread and beside eps: a row of 129 times 1000.1 came out 0.02 from the bias.  (The same for every row costs 7%
    // at 32,768 x 2048 bf16.)  All lanes of a row, and so all wavefronts of a wide one, take one branch.
    if (q[0] * inv < 0x1p-16f * mean * mean) {
      s[0] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s[0] += x[e];
      group_sum<kL, 1>(s, red, turn);
      const float left = s[0] * inv;
      centre(left);
      mean += left;
    }
    const float rstd = 1.0f / sqrtf(q[0] * inv + P.eps);
    T* yr = static_cast<T*>(P.y) + row * w;
    each_vec<V, kL, NV>(l, w, [&](int k, int c, auto whole) {
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = fmaf(x[k * V + e] * rstd, g[k * V + e], b[k * V + e]);
      store_row<T, V>(o, yr, c, w, whole);
    });
    if (P.stats && l == 0) *reinterpret_cast<float2*>(P.stats + 2 * row) = make_float2(mean, rstd);
  }
}

template <typename T, int V, int kL, int NV>
__global__ __launch_bounds__(kL > 64 ? kL : 256) void k_layer_norm_bwd(LnArgs P) {
  constexpr int kR = kL > 64 ? 1 : 256 / kL, E = NV * V;
  __shared__ float red[2][4][16];
  const int l = threadIdx.x % kL, rg = threadIdx.x / kL, w = P.w;
  const float inv = 1.0f / (float)w;
  float g[E], ag[E], ab[E];
  load_params<V, kL, NV>(P.g, P.g_type, l, w, 1.f, g);
#pragma unroll
  for (int e = 0; e < E; ++e) ag[e] = ab[e] = 0.f;
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kR + rg; row < P.n; row += (int64_t)gridDim.x * kR) {
    const T* xr = static_cast<const T*>(P.x) + row * P.ldx;
    const T* gr = static_cast<const T*>(P.gy) + row * P.ldgy;
    const float2 st = *reinterpret_cast<const float2*>(P.stats + 2 * row);
    float xh[E], gy[E], s[2] = {0.f, 0.f};
    RowLoad<T, V, kL, NV> rx, ry;
    rx.load(xr, l, w);
    ry.load(gr, l, w);
    rx.template get<false>(l, w, xh);              // past the row's end gy is zero, and so is all that x enters
    ry.get(l, w, gy);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float h = xh[e] = (xh[e] - st.x) * st.y;
      float& u = gy[e];
      ag[e] = fmaf(u, h, ag[e]);
      ab[e] += u;
      u = rounded_product(u, g[e]);
      s[0] += u;
      s[1] = fmaf(u, h, s[1]);
    }
    group_sum<kL, 2>(s, red, turn);
    const float m1 = s[0] * inv, m2 = s[1] * inv;
    T* o = static_cast<T*>(P.gx) + row * w;
    each_vec<V, kL, NV>(l, w, [&](int k, int c, auto whole) {
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = st.y * (gy[k * V + e] - m1 - xh[k * V + e] * m2);
      store_row<T, V>(v, o, c, w, whole);
    });
  }
  if (P.part) {
    write_part<V, kL, NV>(ag, l, w, P.part + (int64_t)blockIdx.x * w);
    write_part<V, kL, NV>(ab, l, w, P.part + ((int64_t)gridDim.x + blockIdx.x) * w);
  }
}

template <typename T, int V, int kL, int NV>
__global__ __launch_bounds__(kL > 64 ? kL : 256) void k_layer_norm_bwd2(LnArgs P) {
  constexpr int kR = kL > 64 ? 1 : 256 / kL, E = NV * V;
  __shared__ float red[2][4][16];
  const int l = threadIdx.x % kL, rg = threadIdx.x / kL, w = P.w;
  const float inv = 1.0f / (float)w;
  float g[E], qg[E], qb[E], ag[E];
  load_params<V, kL, NV>(P.g, P.g_type, l, w, 1.f, g);
  load_params<V, kL, NV>(P.qg, P.g_type, l, w, 0.f, qg);
  load_params<V, kL, NV>(P.qb, P.b_type, l, w, 0.f, qb);
#pragma unroll
  for (int e = 0; e < E; ++e) ag[e] = 0.f;
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kR + rg; row < P.n; row += (int64_t)gridDim.x * kR) {
    const T* xr = static_cast<const T*>(P.x) + row * P.ldx;
    const T* gr = static_cast<const T*>(P.gy) + row * P.ldgy;
    const T* qr = static_cast<const T*>(P.qx) + row * P.ldq;
    const float2 st = *reinterpret_cast<const float2*>(P.stats + 2 * row);
    const float r = st.y;
    float xh[E], gy[E], q[E];
    float s[4] = {0.f, 0.f, 0.f, 0.f}, squ[1] = {0.f};
    RowLoad<T, V, kL, NV> rx, ry, rq;
    rx.load(xr, l, w);
    ry.load(gr, l, w);
    if (P.qx) rq.load(qr, l, w);
    rx.template get<false>(l, w, xh);              // past the row's end gy, qx, qg and qb are zero
    ry.get(l, w, gy);
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = 0.f;
    if (P.qx) rq.get(l, w, q);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float h = xh[e] = (xh[e] - st.x) * r;
      const float u = gy[e] * g[e], v = q[e];
      s[0] += u;
      s[1] = fmaf(u, h, s[1]);
      s[2] += v;
      s[3] = fmaf(v, h, s[3]);
      squ[0] = fmaf(v, u, squ[0]);
    }
    group_sum<kL, 4>(s, red, turn);
    group_sum<kL, 1>(squ, red, turn);
    const float ub = s[0] * inv, c_ = s[1] * inv, qm = s[2] * inv, m = s[3] * inv;
    const float rr = r * r * (squ[0] * inv - qm * ub - c_ * m);      // r <qx gx>
    float t[2] = {0.f, 0.f};
    T* o1 = static_cast<T*>(P.y) + row * w;
    each_vec<V, kL, NV>(l, w, [&](int k, int c, auto whole) {
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int i = k * V + e;
        const float a = r * (q[i] - qm - xh[i] * m);
        v[e] = g[i] * a + qg[i] * xh[i] + qb[i];
        ag[i] = fmaf(gy[i], a, ag[i]);
        const float x = qg[i] * gy[i] - r * (c_ * q[i] + m * gy[i] * g[i]);
        q[i] = x;
        t[0] += x;
        t[1] = fmaf(x, xh[i], t[1]);
      }
      store_row<T, V>(v, o1, c, w, whole);
    });
    group_sum<kL, 2>(t, red, turn);
    const float mx = t[0] * inv, mxx = t[1] * inv;
    T* o2 = static_cast<T*>(P.gx) + row * w;
    each_vec<V, kL, NV>(l, w, [&](int k, int c, auto whole) {
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = r * (q[k * V + e] - mx - xh[k * V + e] * mxx) - rr * xh[k * V + e];
      store_row<T, V>(v, o2, c, w, whole);
    });
  }
  if (P.part) write_part<V, kL, NV>(ag, l, w, P.part + (int64_t)blockIdx.x * w);
}

// out_a[c] = the sum over the n_part rows of part [a][n_part][w], a = blockIdx.y: 32 lanes take every 32nd row, then
// a tree; rounded once to the parameter's type.
__global__ __launch_bounds__(1024) void k_layer_norm_params(const float* __restrict__ part, int n_part, int w,
                                                            void* out0, int type0, void* out1, int type1) {
  __shared__ float red[32][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), r = threadIdx.x >> 5;
  const float* p = part + (int64_t)blockIdx.y * n_part * w;
  float s = 0.f;
  if (c < w) {
#pragma unroll 8
    for (int i = r; i < n_part; i += 32) s += p[(int64_t)i * w + c];
  }
  red[r][threadIdx.x & 31] = s;
  __syncthreads();
  if (r == 0 && c < w) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += red[i][threadIdx.x];
    void* out = blockIdx.y ? out1 : out0;
    const int type = blockIdx.y ? type1 : type0;
    if (!out) return;
    if (type == E2V2_F32) static_cast<float*>(out)[c] = s;
    else if (type == E2V2_BF16) static_cast<__bf16*>(out)[c] = (__bf16)s;
    else static_cast<_Float16*>(out)[c] = (_Float16)s;
  }
}

enum class LnPass { kFwd, kBwd, kBwd2 };

template <LnPass kPass, typename T, int V, int kL, int NV>
void ln_launch(const LnArgs& P, unsigned grid, hipStream_t s) {
  const dim3 block(kL > 64 ? kL : 256);
  if constexpr (kPass == LnPass::kFwd)
    hipLaunchKernelGGL((k_layer_norm_fwd<T, V, kL, NV>), dim3(grid), block, 0, s, P);
  else if constexpr (kPass == LnPass::kBwd)
    hipLaunchKernelGGL((k_layer_norm_bwd<T, V, kL, NV>), dim3(grid), block, 0, s, P);
  else
    hipLaunchKernelGGL((k_layer_norm_bwd2<T, V, kL, NV>), dim3(grid), block, 0, s, P);
}

template <LnPass kPass, typename T>
void ln_dispatch(const LnArgs& P, unsigned grid, hipStream_t s) {
  constexpr int V = RowVec<T>::n;
  constexpr bool kBwd = kPass == LnPass::kBwd;
  const RowShape f = row_shape(P.w, V, kBwd);
  switch (f.lanes * 16 + f.vecs) {
    case 2 * 16: return ln_launch<kPass, T, 1, 2, 1>(P, grid, s);
    case 4 * 16: return ln_launch<kPass, T, 1, 4, 1>(P, grid, s);
    case 8 * 16: return ln_launch<kPass, T, 1, 8, 1>(P, grid, s);
    case 2 * 16 + 1: return ln_launch<kPass, T, V, 2, 1>(P, grid, s);
    case 4 * 16 + 1: return ln_launch<kPass, T, V, 4, 1>(P, grid, s);
    case 8 * 16 + 1: return ln_launch<kPass, T, V, 8, 1>(P, grid, s);
    case 16 * 16 + 1: return ln_launch<kPass, T, V, 16, 1>(P, grid, s);
    case 32 * 16 + 1: return ln_launch<kPass, T, V, 32, 1>(P, grid, s);
    case 4 * 16 + 3: return ln_launch<kPass, T, V, 4, 3>(P, grid, s);
    case 8 * 16 + 3: return ln_launch<kPass, T, V, 8, 3>(P, grid, s);
    case 16 * 16 + 3: return ln_launch<kPass, T, V, 16, 3>(P, grid, s);
    case 64 * 16 + 1: return ln_launch<kPass, T, V, 64, 1>(P, grid, s);
    case 32 * 16 + 3: return ln_launch<kPass, T, V, 32, 3>(P, grid, s);
    case 64 * 16 + 2: return ln_launch<kPass, T, V, 64, 2>(P, grid, s);
  }
  if constexpr (V == 4) {
    switch (f.lanes * 16 + f.vecs) {
      case 64 * 16 + 3: return ln_launch<kPass, T, V, 64, 3>(P, grid, s);
      case 64 * 16 + 4: return ln_launch<kPass, T, V, 64, 4>(P, grid, s);
      case 256 * 16 + 8:
        if constexpr (!kBwd) return ln_launch<kPass, T, V, 256, 8>(P, grid, s);
    }
  }
  switch (f.lanes * 16 + f.vecs) {
    case 256 * 16 + 1:
      if constexpr (V == 8) return ln_launch<kPass, T, V, 256, 1>(P, grid, s);
      break;
    case 256 * 16 + 2: return ln_launch<kPass, T, V, 256, 2>(P, grid, s);
    case 256 * 16 + 3: return ln_launch<kPass, T, V, 256, 3>(P, grid, s);
    case 256 * 16 + 4:
      if constexpr (!kBwd || V == 4) return ln_launch<kPass, T, V, 256, 4>(P, grid, s);
      break;
    case 1024 * 16 + 8 / V:
      if constexpr (kBwd) return ln_launch<kPass, T, V, 1024, 8 / V>(P, grid, s);
      break;
    default: return ln_launch<kPass, T, V, 1024, 16 / V>(P, grid, s);
  }
}

template <LnPass kPass>
void ln_run(const LnArgs& P, int type, unsigned grid, hipStream_t s) {
  if (type == E2V2_F32) ln_dispatch<kPass, float>(P, grid, s);
  else if (type == E2V2_BF16) ln_dispatch<kPass, __bf16>(P, grid, s);
  else ln_dispatch<kPass, _Float16>(P, grid, s);
}

// Workgroups of a pass.  They stride over the rows, with the parameters loaded once: a workgroup for every few rows
// loads them again each time (forward, 127,113 x 128 fp32: 26 us with 1,024 workgroups, 38 with one for 8 rows; 32,768
// x 2048 bf16: 51 with 2,048, 232 with one a row).  Where sums of the parameters are left, fewer partial rows are
// fewer bytes, but one vector a lane needs four workgroups a CU to have enough loads in flight (200,000 x 256 bf16: 60
// us with 1,024, 83 with 512; 60,000 x 512 fp32, two vectors: 76 and 72; 6,007 x 5001 fp32, 1024 lanes: 99 and, with
// 256, 81).  Without sums and with narrow rows the backward pass only reloads the weight, which the caches hold: one
// row a lane group (853,991 x 128 fp32: 215 us, 244 with 1,024).
unsigned ln_grid(const LnArgs& P, int type, LnPass pass, bool sums) {
  const int v = 16 / type_size(type);
  const RowShape f = row_shape(P.w, v, pass == LnPass::kBwd);
  const int r = f.lanes > 64 ? 1 : 256 / f.lanes;
  int64_t most = f.lanes == 1024 ? 512 : f.lanes == 256 ? 2048 : 1024;
  if (sums) most = f.lanes == 1024 ? 256 : f.vecs <= 1 ? 1024 : 512;
  else if (pass != LnPass::kFwd && f.lanes <= 32 && f.vecs <= 1) most = 1 << 23;
  return (unsigned)std::min<int64_t>((P.n + r - 1) / r, most);
}

int ln_check(const char* what, const e2v2_layer_norm_args* a, bool bwd, bool bwd2) {
  E2V2_REQUIRE(a, "%s: null arguments", what);
  E2V2_REQUIRE(a->n >= 0 && a->w > 0 && a->w <= kLnMaxWidth, "%s: %lld rows of width %d (1 to %d)", what,
               (long long)a->n, a->w, kLnMaxWidth);
  E2V2_REQUIRE(type_ok(a->type) && type_ok(a->g_type) && type_ok(a->b_type), "%s: types %d, %d, %d", what, a->type,
               a->g_type, a->b_type);
  E2V2_REQUIRE(a->ldx >= 0 && a->ldgy >= 0 && a->ldqx >= 0, "%s: negative row stride", what);
  const uintptr_t all = (uintptr_t)a->x | (uintptr_t)a->gy | (uintptr_t)a->qx | (uintptr_t)a->y | (uintptr_t)a->gx;
  E2V2_REQUIRE(all % type_size(a->type) == 0 && (uintptr_t)a->stats % 8 == 0, "%s: misaligned operand", what);
  if (a->n == 0) return 0;
  E2V2_REQUIRE(a->x && (bwd || a->y) && (!bwd || (a->gy && a->stats && a->gx)) && (!bwd2 || a->y),
               "%s: null operand", what);
  return 0;
}

LnArgs ln_args(const e2v2_layer_norm_args* a) {
  return LnArgs{a->x, a->gy, a->qx, a->g, a->b, a->qg, a->qb, a->y, a->gx, a->stats, nullptr, a->n, a->ldx, a->ldgy,
                a->ldqx, a->w, a->g_type, a->b_type, a->eps};
}

}  // namespace

int launch_param_sums(const float* part, int n_part, int w, int arrays, void* o0, int t0, void* o1, int t1,
                      hipStream_t s) {
  hipLaunchKernelGGL(k_layer_norm_params, dim3((w + 31) / 32, arrays), dim3(1024), 0, s, part, n_part, w, o0, t0, o1,
                     t1);
  E2V2_LAUNCHED("k_layer_norm_params");
  return 0;
}
}  // namespace e2v2

using namespace e2v2;

E2V2_API int e2v2_layer_norm_fwd(const e2v2_layer_norm_args* a, hipStream_t s) {
  if (const int rc = ln_check("layer_norm_fwd", a, false, false)) return rc;
  if (a->n == 0) return 0;
  LnArgs P = ln_args(a);
  P.gy = P.qx = P.gx = nullptr;
  P.ldgy = P.ldq = 0;
  ln_run<LnPass::kFwd>(P, a->type, ln_grid(P, a->type, LnPass::kFwd, false), s);
  E2V2_LAUNCHED("k_layer_norm_fwd");
  return 0;
}

E2V2_API int64_t e2v2_layer_norm_workspace(int64_t n, int w) {
  if (n <= 0 || w <= 0) return 0;
  return 2 * std::min<int64_t>(n, kLnMaxParts) * w * 4;
}

E2V2_API int e2v2_layer_norm_bwd(const e2v2_layer_norm_args* a, void* gg, void* gb, float* ws, int64_t ws_bytes,
                                 hipStream_t s) {
  if (const int rc = ln_check("layer_norm_bwd", a, true, false)) return rc;
  const bool params = gg || gb;
  E2V2_REQUIRE(!params || (ws_bytes >= e2v2_layer_norm_workspace(a->n, a->w) && (ws || a->n == 0)),
               "layer_norm_bwd: workspace of %lld bytes", (long long)ws_bytes);
  LnArgs P = ln_args(a);
  P.qx = P.y = nullptr;
  P.ldq = 0;
  P.part = params ? ws : nullptr;
  const unsigned grid = ln_grid(P, a->type, LnPass::kBwd, params);
  if (grid) {
    ln_run<LnPass::kBwd>(P, a->type, grid, s);
    E2V2_LAUNCHED("k_layer_norm_bwd");
  }
  return params ? launch_param_sums(ws, (int)grid, a->w, 2, gg, a->g_type, gb, a->b_type, s) : 0;
}

E2V2_API int e2v2_layer_norm_bwd2(const e2v2_layer_norm_args* a, void* gg, float* ws, int64_t ws_bytes,
                                  hipStream_t s) {
  if (const int rc = ln_check("layer_norm_bwd2", a, true, true)) return rc;
  E2V2_REQUIRE(!gg || (ws_bytes >= e2v2_layer_norm_workspace(a->n, a->w) && (ws || a->n == 0)),
               "layer_norm_bwd2: workspace of %lld bytes", (long long)ws_bytes);
  LnArgs P = ln_args(a);
  P.part = gg ? ws : nullptr;
  const unsigned grid = ln_grid(P, a->type, LnPass::kBwd2, gg != nullptr);
  if (grid) {
    ln_run<LnPass::kBwd2>(P, a->type, grid, s);
    E2V2_LAUNCHED("k_layer_norm_bwd2");
  }
  return gg ? launch_param_sums(ws, (int)grid, a->w, 1, gg, a->g_type, nullptr, 0, s) : 0;
}
