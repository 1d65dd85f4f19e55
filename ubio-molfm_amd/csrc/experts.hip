// Products grouped by expert in fp32, bf16 and fp16 (mm.h): rows offsets[e] .. offsets[e + 1] belong to expert e, and
//   forward          y[t] = W[e] x[t]              W [experts][n][k], read as it lies
//   rows' gradient   gx[t] = W[e]^T gy[t]          W read along its columns
//   weights' grad.   gW[e] = sum_t gy[t] x[t]^T    both operands read along their columns, over ragged rows
// Rows of no expert give zeros.
//
// 16,384 rows over 32 experts of 1408 x 2048 bf16, operands in turn: 118, 121 and 139 us (95 GFLOP each; the weights' gradient
// writes 184 MB), unevenly 124, 123 and 145; where rows start off 16 bytes (1408 x 2047) 260, 253 and 345.  10,000 rows over 6 of 256 x 256 fp32: 21, 21 and 26.
#include <algorithm>

#include "mm.h"

namespace e2v2 {
namespace {

// The parts that the rows of each expert are cut into for the weights' gradient: enough workgroups for the 256 CUs where
// experts and tiles are few (one expert of 16,384 rows, 1536 x 2048 bf16: 131 us, uncut 162).
int splits_of(int64_t rows, int64_t n, int64_t k, int groups) {
  const int64_t tiles = groups * ((n + 127) / 128) * ((k + 127) / 128);
  if (tiles >= (rows / groups >= 4096 ? 257 : 192)) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>({512 / tiles, rows / groups / 256, 16}));
}

template <int kT, bool kAO, bool kBO, int kGroup, bool kStaged>
void run(const MmArgs& P, hipStream_t s) {
  if constexpr (!kStaged) {
    if constexpr (!kAO && !kBO) {
      if (thin_rows(P.m, P.n, (int64_t)P.k * elem_size(kT), P.groups)) return launch_thin<kT, kGroup>(P, s);
    }
    // Tiles of 256 where they fill the 256 CUs and an expert has rows for several of them (32 experts of 512 rows, 1408 x
    // 2048 bf16, forward and both gradients: 134, 133 and 137 us, with tiles of 128 131, 120 and 129; 16 of 2048 rows, 2048 x
    // 2048: 280, 289 and 254, and 306, 301 and 295); of 64 where not even those of 128 fill them (8 experts of 62 rows,
    // 512 x 1024 bf16: 11 us, 14).
    const int64_t rows = kGroup == kRed ? P.k : P.m, each = rows / P.groups;
    auto tiles = [&](int64_t t) {
      return (kGroup == kRed ? P.groups * ((P.m + t - 1) / t) : P.m / t + std::min(P.groups, P.m)) * ((P.n + t - 1) / t);
    };
    if constexpr (kT != kF32) {
      if (tiles(256) >= 200 && each >= (P.groups > 1 ? 1024 : 192))
        return launch_mm<kT, kAO, kBO, 256, 256, 2, 4, kGroup, false>(P, s);
    }
    if (tiles(128) * P.splits < 256) return launch_mm<kT, kAO, kBO, 64, 64, 2, 1, kGroup, false>(P, s);
  }
  launch_mm<kT, kAO, kBO, 128, 128, 2, 2, kGroup, kStaged>(P, s);
}

template <int kT>
void run_pass(const MmArgs& P, int pass, bool staged, hipStream_t s) {
  if (pass == E2V2_EXPERT_FORWARD)
    staged ? run<kT, false, false, kRows, true>(P, s) : run<kT, false, false, kRows, false>(P, s);
  else if (pass == E2V2_EXPERT_ROWS)
    staged ? run<kT, false, true, kRows, true>(P, s) : run<kT, false, true, kRows, false>(P, s);
  else
    staged ? run<kT, true, true, kRed, true>(P, s) : run<kT, true, true, kRed, false>(P, s);
}

}  // namespace
}  // namespace e2v2

using namespace e2v2;

E2V2_API int64_t e2v2_expert_product_workspace(int64_t rows, int64_t n, int64_t k, int experts) {
  if (rows <= 0 || n <= 0 || k <= 0 || experts <= 0) return 0;
  const int splits = splits_of(rows, n, k, experts);
  return splits > 1 ? splits * experts * n * k * 4 : 0;
}

E2V2_API int e2v2_expert_product(const e2v2_expert_args* a, int pass, float* ws, int64_t ws_bytes, hipStream_t s) {
  E2V2_REQUIRE(a, "expert_product: null arguments");
  E2V2_REQUIRE(pass >= E2V2_EXPERT_FORWARD && pass <= E2V2_EXPERT_WEIGHTS, "expert_product: pass %d", pass);
  E2V2_REQUIRE(a->rows >= 0 && a->n >= 0 && a->k >= 0 && a->rows <= INT32_MAX / 2 && a->n <= INT32_MAX / 2 &&
                   a->k <= INT32_MAX / 2 && a->experts > 0, "expert_product: %lld rows, %d experts of %lld x %lld",
               (long long)a->rows, a->experts, (long long)a->n, (long long)a->k);
  E2V2_REQUIRE(a->type >= E2V2_F32 && a->type <= E2V2_F16, "expert_product: type %d", a->type);
  const int size = a->type == E2V2_F32 ? 4 : 2;
  // rows [T][..] of each pass, its product's extents and its operands
  const bool fwd = pass == E2V2_EXPERT_FORWARD, wgrad = pass == E2V2_EXPERT_WEIGHTS;
  MmArgs P{};
  P.m = (int)(wgrad ? a->n : a->rows);
  P.n = (int)(fwd ? a->n : a->k);
  P.k = (int)(fwd ? a->k : wgrad ? a->rows : a->n);
  if (P.m == 0 || P.n == 0) return 0;
  const void* pa = fwd ? a->x : a->gy;
  const void* pb = wgrad ? a->x : a->w;
  const int64_t lda = fwd ? a->ldx : a->ldgy, ldb = wgrad ? a->ldx : a->ldw;
  E2V2_REQUIRE(a->y && a->offsets && (a->rows == 0 || P.k == 0 || (pa && pb)), "expert_product: null operand");
  const int64_t wide = (fwd || wgrad ? a->k : 0), wide_gy = fwd ? 0 : a->n;
  E2V2_REQUIRE(a->ldx >= wide && a->ldgy >= wide_gy && (wgrad || a->ldw >= a->k) && a->ldy >= P.n &&
                   lda <= kMaxPitch / size && ldb <= kMaxPitch / size, "expert_product: row strides %lld, %lld, %lld, %lld",
               (long long)a->ldx, (long long)a->ldw, (long long)a->ldgy, (long long)a->ldy);
  E2V2_REQUIRE(((uintptr_t)pa | (uintptr_t)pb | (uintptr_t)a->y) % size == 0 && (uintptr_t)a->offsets % 4 == 0 &&
                   (uintptr_t)ws % 16 == 0, "expert_product: misaligned operand");
  P.a = static_cast<const uint8_t*>(pa);
  P.b = static_cast<const uint8_t*>(pb);
  P.y = a->y;
  P.part = ws;
  P.offsets = a->offsets;
  P.lda = lda * size;
  P.ldb = ldb * size;
  P.b_group = a->w_group * size;
  P.ldy = a->ldy;
  P.groups = a->experts;
  P.out_type = a->type;
  P.fill = a->fill;
  P.splits = wgrad ? splits_of(a->rows, a->n, a->k, a->experts) : 1;
  E2V2_REQUIRE(P.splits == 1 || (ws && ws_bytes >= e2v2_expert_product_workspace(a->rows, a->n, a->k, a->experts)),
               "expert_product: workspace of %lld bytes", (long long)ws_bytes);
  const int64_t tiles = wgrad ? (int64_t)a->experts * ((P.m + 63) / 64) * ((P.n + 63) / 64)
                              : (a->rows / 16 + a->experts) * ((P.n + 15) / 16);
  E2V2_REQUIRE(tiles < INT32_MAX / 2, "expert_product: %lld tiles", (long long)tiles);
  const bool staged = ((uintptr_t)pa | (uintptr_t)pb | (uintptr_t)P.lda | (uintptr_t)P.ldb |
                       (uintptr_t)(wgrad ? 0 : P.b_group)) % 16 != 0;
  if (a->type == E2V2_F32) run_pass<kF32>(P, pass, staged, s);
  else if (a->type == E2V2_BF16) run_pass<kBf16>(P, pass, staged, s);
  else run_pass<kF16>(P, pass, staged, s);
  E2V2_LAUNCHED("k_mm");
  if (P.splits > 1) {
    launch_mm_sum(P, (int64_t)P.groups * P.m, s);
    E2V2_LAUNCHED("k_mm_sum");
  }
  return 0;
}
