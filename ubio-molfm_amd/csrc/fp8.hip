// Rows and weights in 8 bits with block scales (quant8.h has the format): quantisation of rows (1 x 128 blocks), of
// weights (128 x 128 tiles) and of the transposes that the gradients' products read, and the values of codes.  Products
// are in mm.h.
//
// Each element is read once: a block's largest value, its scale and its codes come from registers.  Bound: HBM.  16384 x
// 4096 bf16, four tensors in turn (a copy reaches 5 TB/s): rows 33 us (6.1 TB/s, two thirds of them reads), values back to
// bf16 33, tiles 45 (4.5), rows along both directions 66 (4.1: a workgroup loads a tile, meets four barriers, stores and
// ends).  One tensor again and again, partly from the cache: 30, 31, 35 and 56.
#include "quant8.h"
#include "rows.h"

namespace e2v2 {
namespace {

struct QuantArgs {
  const void* x; uint8_t* codes; uint8_t* scales; uint8_t* codes_t; uint8_t* scales_t;
  int64_t ldx, ldc, ldt, x_batch, c_batch, s_batch, t_batch, st_batch;
  int n, w;
};

// The 8 elements of a row from column c on; zeros behind its end.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int c, int w, float (&v)[8]) {
  constexpr int V = RowVec<T>::n;
  if (c + 8 <= w) {
#pragma unroll
    for (int k = 0; k < 8; k += V) {
      const auto f = __builtin_convertvector(*reinterpret_cast<const typename RowVec<T>::any*>(row + c + k),
                                             typename RowVec<T>::ftype);
#pragma unroll
      for (int e = 0; e < V; ++e) v[k + e] = f[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < w ? (float)row[c + e] : 0.f;
  }
}

__device__ __forceinline__ uint2 codes8(const float (&v)[8], float up) {
  return make_uint2(codes4(v[0] * up, v[1] * up, v[2] * up, v[3] * up), codes4(v[4] * up, v[5] * up, v[6] * up, v[7] * up));
}

// 16 lanes a block of 128 columns.  Rows of codes lie a multiple of 16 bytes apart; their padding gets zeros.
template <typename T>
__global__ __launch_bounds__(256) void k_quant_rows(QuantArgs P) {
  const unsigned nb = (unsigned)(P.w + kBlock8 - 1) / kBlock8, total = (unsigned)P.n * nb;
  const int l = threadIdx.x & 15;
  for (unsigned i = blockIdx.x * 16 + (threadIdx.x >> 4); i < total; i += gridDim.x * 16) {
    const unsigned row = i / nb, b = i - row * nb;
    const int c = (int)b * kBlock8 + l * 8;
    float v[8];
    load8(static_cast<const T*>(P.x) + (int64_t)row * P.ldx, c, P.w, v);
    const int s = scale_byte(top_bits([&](auto bits) {
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, bits(v[e]));
      return lanes_max<16>(m);
    }));
    if (c < P.ldc) *reinterpret_cast<uint2*>(P.codes + (int64_t)row * P.ldc + c) = codes8(v, scale_up(s));
    if (l == 0) P.scales[(int64_t)b * P.n + row] = (uint8_t)s;
  }
}

// One tile of 128 x 128, thread (r, l) holding rows 8 r .. 8 r + 7 and columns 8 l .. 8 l + 7.  kTile: one scale for the
// tile, codes and codes_t (either may be NULL) the same values; else codes with a scale for each row of the tile and
// codes_t with one for each column.  The transpose goes through LDS: column j's 128 codes are one row there, its 8-byte
// pieces moved round by j / 8, so that the 16 lanes that write pieces of 16 columns do not meet in one bank.
// bits: of the values' magnitudes; all: the largest in the tile, or kInfBits where some are not finite.
template <bool kTile, typename Bits>
__device__ __forceinline__ void quant_tile(const QuantArgs& P, const float (&v)[8][8], uint32_t (*most)[kBlock8],
                                           uint8_t (*turned)[kBlock8], Bits bits, uint32_t all) {
  const int l = threadIdx.x & 15, r = threadIdx.x >> 4, wv = threadIdx.x >> 6;
  const int r0 = blockIdx.y * kBlock8 + r * 8, c0 = blockIdx.x * kBlock8, c = c0 + l * 8;
  const int64_t z = blockIdx.z;
  float up[8];                                     // of the thread's rows, then of its columns
  const int nb = (P.w + kBlock8 - 1) / kBlock8, nbt = (P.n + kBlock8 - 1) / kBlock8;
  if constexpr (kTile) {
    if (all >= kInfBits) {
      uint32_t m = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, bits(v[k][e]));
      m = lanes_max<64>(m);
      if ((threadIdx.x & 63) == 0) most[wv][0] = m;
      __syncthreads();
      all = max(max(most[0][0], most[1][0]), max(most[2][0], most[3][0]));
    }
    const int s = scale_byte(all);
    if (threadIdx.x == 0) {
      if (P.scales) P.scales[z * P.s_batch + (int64_t)blockIdx.y * nb + blockIdx.x] = (uint8_t)s;
      if (P.scales_t) P.scales_t[z * P.st_batch + (int64_t)blockIdx.x * nbt + blockIdx.y] = (uint8_t)s;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) up[k] = scale_up(s);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, bits(v[k][e]));
      const int s = scale_byte(lanes_max<16>(m));
      up[k] = scale_up(s);
      if (P.scales && l == 0 && r0 + k < P.n) P.scales[(int64_t)blockIdx.x * P.n + r0 + k] = (uint8_t)s;
    }
  }
  if (P.codes) {
    uint8_t* q = P.codes + z * P.c_batch;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (r0 + k < P.n && c < P.ldc) *reinterpret_cast<uint2*>(q + (int64_t)(r0 + k) * P.ldc + c) = codes8(v[k], up[k]);
  }
  if (!P.codes_t) return;                          // the same for the whole workgroup
  if constexpr (!kTile) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t m = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) m = max(m, bits(v[k][e]));
      auto a = __builtin_amdgcn_permlane16_swap(m, m, false, false);
      m = max((uint32_t)a[0], (uint32_t)a[1]);
      a = __builtin_amdgcn_permlane32_swap(m, m, false, false);
      m = max((uint32_t)a[0], (uint32_t)a[1]);
      if ((threadIdx.x & 63) < 16) most[wv][l * 8 + e] = m;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = l * 8 + e;
      const int s = scale_byte(max(max(most[0][j], most[1][j]), max(most[2][j], most[3][j])));
      up[e] = scale_up(s);
      if (r == 0 && c + e < P.w) P.scales_t[(int64_t)blockIdx.y * P.w + c + e] = (uint8_t)s;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float t[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = v[k][e];
    *reinterpret_cast<uint2*>(&turned[l * 8 + e][((r + l) & 15) * 8]) = codes8(t, up[e]);
  }
  __syncthreads();
  uint8_t* q = P.codes_t + z * P.t_batch;
  for (int i = threadIdx.x; i < kBlock8 * 16; i += 256) {
    const int j = i >> 4, p = i & 15, at = blockIdx.y * kBlock8 + p * 8;
    if (c0 + j < P.w && at < P.ldt)
      *reinterpret_cast<uint2*>(q + (int64_t)(c0 + j) * P.ldt + at) =
          *reinterpret_cast<const uint2*>(&turned[j][((p + (j >> 3)) & 15) * 8]);
  }
}

template <typename T, bool kTile>
__global__ __launch_bounds__(256) void k_quant_tiles(QuantArgs P) {
  __shared__ uint32_t most[4][kBlock8];
  __shared__ __attribute__((aligned(16))) uint8_t turned[kBlock8][kBlock8];
  const int l = threadIdx.x & 15, r = threadIdx.x >> 4, wv = threadIdx.x >> 6;
  const int r0 = blockIdx.y * kBlock8 + r * 8, c0 = blockIdx.x * kBlock8, c = c0 + l * 8;
  const T* x = static_cast<const T*>(P.x) + blockIdx.z * P.x_batch;
  float v[8][8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (r0 + k < P.n) {
      load8(x + (int64_t)(r0 + k) * P.ldx, c, P.w, v[k]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[k][e] = 0.f;
    }
  }
  // whether a value of the tile is not finite, and the function of those left that is taken
  uint32_t all = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) all = max(all, abs_bits(v[k][e]));
  all = lanes_max<64>(all);
  if ((threadIdx.x & 63) == 0) most[wv][0] = all;
  __syncthreads();
  all = max(max(most[0][0], most[1][0]), max(most[2][0], most[3][0]));
  __syncthreads();
  if (all < kInfBits) quant_tile<kTile>(P, v, most, turned, [](float x) { return abs_bits(x); }, all);
  else quant_tile<kTile>(P, v, most, turned, [](float x) { return finite_bits(x); }, kInfBits);
}

struct ValueArgs {
  const uint8_t* codes; const uint8_t* scales; void* out;
  int64_t ldc, s_ld, s_k;
  int n, w, block_rows, rows_each;     // rows_each: rows of one of several weights
  bool aligned;
};

// Values of codes: 16 lanes a block of 128 columns, 8 codes a lane.
template <typename T>
__global__ __launch_bounds__(256) void k_values8(ValueArgs P) {
  const unsigned nb = (unsigned)(P.w + kBlock8 - 1) / kBlock8, total = (unsigned)P.n * nb;
  const int l = threadIdx.x & 15;
  for (unsigned i = blockIdx.x * 16 + (threadIdx.x >> 4); i < total; i += gridDim.x * 16) {
    const unsigned row = i / nb, b = i - row * nb;
    const int c = (int)b * kBlock8 + l * 8;
    if (c >= P.w) continue;
    unsigned srow = row;
    if (P.block_rows > 1) {
      const unsigned each = (unsigned)P.rows_each, of = row / each;
      srow = of * ((each + kBlock8 - 1) / kBlock8) + (row - of * each) / kBlock8;
    }
    const float s = scale_value(P.scales[(int64_t)srow * P.s_ld + (int64_t)b * P.s_k]);
    const uint8_t* q = P.codes + (int64_t)row * P.ldc + c;
    uint2 u = make_uint2(0, 0);
    if (P.aligned && c + 8 <= P.w) {
      u = *reinterpret_cast<const uint2*>(q);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t v = c + e < P.w ? q[e] : 0;
        if (e < 4) u.x |= v << (8 * e);
        else u.y |= v << (8 * (e - 4));
      }
    }
    float v[8];
    auto two = [&](uint32_t d, float* o) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)d, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)d, true);
      o[0] = lo[0] * s, o[1] = lo[1] * s, o[2] = hi[0] * s, o[3] = hi[1] * s;
    };
    two(u.x, v);
    two(u.y, v + 4);
    T* o = static_cast<T*>(P.out) + (int64_t)row * P.w;
    constexpr int V = RowVec<T>::n;
#pragma unroll
    for (int k = 0; k < 8; k += V) store_row<T, V>(v + k, o, c + k, P.w, false);
  }
}

unsigned row_blocks(int64_t total) { return (unsigned)(total < 16 * 8192 ? (total + 15) / 16 : 8192); }

}  // namespace
}  // namespace e2v2

using namespace e2v2;

E2V2_API int e2v2_quantize8(const e2v2_quantize8_args* a, hipStream_t s) {
  E2V2_REQUIRE(a, "quantize8: null arguments");
  E2V2_REQUIRE(type_ok(a->type) && a->mode >= 0 && a->mode <= 2, "quantize8: type %d, mode %d", a->type, a->mode);
  E2V2_REQUIRE(a->n >= 0 && a->width >= 0 && a->batch >= 0 && a->n <= INT32_MAX && a->width <= INT32_MAX,
               "quantize8: %lld x %lld, %d of them", (long long)a->n, (long long)a->width, a->batch);
  if (a->n == 0 || a->width == 0 || a->batch == 0) return 0;
  const int64_t nb = (a->width + kBlock8 - 1) / kBlock8, nbt = (a->n + kBlock8 - 1) / kBlock8;
  E2V2_REQUIRE(a->x && (uintptr_t)a->x % type_size(a->type) == 0, "quantize8: null or misaligned operand");
  E2V2_REQUIRE(!a->codes || (a->scales && a->ldc >= a->width && a->ldc % 16 == 0 && (uintptr_t)a->codes % 16 == 0),
               "quantize8: rows of codes lie a multiple of 16 bytes apart, got %lld", (long long)a->ldc);
  E2V2_REQUIRE(!a->codes_t || (a->scales_t && a->ldt >= a->n && a->ldt % 16 == 0 && (uintptr_t)a->codes_t % 16 == 0),
               "quantize8: rows of transposed codes lie a multiple of 16 bytes apart, got %lld", (long long)a->ldt);
  QuantArgs P{a->x, a->codes, a->scales, a->codes_t, a->scales_t, a->ldx, a->ldc, a->ldt, a->x_batch,
              a->n * a->ldc, nbt * nb, a->width * a->ldt, nbt * nb, (int)a->n, (int)a->width};
  if (a->mode == E2V2_QUANT_ROWS) {
    E2V2_REQUIRE(a->codes && !a->codes_t && a->batch == 1, "quantize8: rows have codes, no transpose and no batch");
    E2V2_REQUIRE(a->n * nb < INT32_MAX, "quantize8: %lld blocks", (long long)(a->n * nb));
    const dim3 grid(row_blocks(a->n * nb));
    if (a->type == E2V2_F32) hipLaunchKernelGGL(k_quant_rows<float>, grid, dim3(256), 0, s, P);
    else if (a->type == E2V2_BF16) hipLaunchKernelGGL(k_quant_rows<__bf16>, grid, dim3(256), 0, s, P);
    else hipLaunchKernelGGL(k_quant_rows<_Float16>, grid, dim3(256), 0, s, P);
    E2V2_LAUNCHED("k_quant_rows");
    return 0;
  }
  E2V2_REQUIRE(a->codes || a->codes_t, "quantize8: no output");
  E2V2_REQUIRE(nbt <= 65535 && a->batch <= 65535, "quantize8: %lld rows, %d weights", (long long)a->n, a->batch);
  E2V2_REQUIRE(a->mode == E2V2_QUANT_TILES || a->batch == 1, "quantize8: both directions of one matrix, got %d", a->batch);
  const dim3 grid((unsigned)nb, (unsigned)nbt, (unsigned)a->batch);
  auto run = [&](auto tile) {
    constexpr bool kTile = decltype(tile)::value;
    if (a->type == E2V2_F32) hipLaunchKernelGGL((k_quant_tiles<float, kTile>), grid, dim3(256), 0, s, P);
    else if (a->type == E2V2_BF16) hipLaunchKernelGGL((k_quant_tiles<__bf16, kTile>), grid, dim3(256), 0, s, P);
    else hipLaunchKernelGGL((k_quant_tiles<_Float16, kTile>), grid, dim3(256), 0, s, P);
  };
  if (a->mode == E2V2_QUANT_TILES) run(std::true_type{});
  else run(std::false_type{});
  E2V2_LAUNCHED("k_quant_tiles");
  return 0;
}

E2V2_API int e2v2_values8(const uint8_t* codes, int64_t ldc, const uint8_t* scales, int64_t s_ld, int64_t s_k, int tiles,
                          int64_t n, int64_t width, int64_t rows_each, void* out, int type, hipStream_t s) {
  E2V2_REQUIRE(type_ok(type), "values8: type %d", type);
  E2V2_REQUIRE(n >= 0 && width >= 0 && width <= INT32_MAX && n <= INT32_MAX && ldc >= 0 && s_ld >= 0 && s_k >= 0,
               "values8: %lld x %lld", (long long)n, (long long)width);
  if (n == 0 || width == 0) return 0;
  const int64_t nb = (width + kBlock8 - 1) / kBlock8;
  E2V2_REQUIRE(codes && scales && out && (uintptr_t)out % type_size(type) == 0, "values8: null or misaligned operand");
  E2V2_REQUIRE(!tiles || (rows_each > 0 && n % rows_each == 0), "values8: %lld rows of weights of %lld", (long long)n,
               (long long)rows_each);
  E2V2_REQUIRE(n * nb < INT32_MAX, "values8: %lld blocks", (long long)(n * nb));
  const ValueArgs P{codes, scales, out, ldc, s_ld, s_k, (int)n, (int)width, tiles ? kBlock8 : 1, (int)(tiles ? rows_each : n),
                    ldc % 8 == 0 && (uintptr_t)codes % 8 == 0};
  const dim3 grid(row_blocks(n * nb));
  if (type == E2V2_F32) hipLaunchKernelGGL(k_values8<float>, grid, dim3(256), 0, s, P);
  else if (type == E2V2_BF16) hipLaunchKernelGGL(k_values8<__bf16>, grid, dim3(256), 0, s, P);
  else hipLaunchKernelGGL(k_values8<_Float16>, grid, dim3(256), 0, s, P);
  E2V2_LAUNCHED("k_values8");
  return 0;
}
