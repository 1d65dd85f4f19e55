// Products of 8-bit rows and 8-bit weights with block scales, dense or with a weight for each expert (mm.h).  The scales
// are powers of two that the matrix instruction applies itself: v_mfma_scale_f32_16x16x128_f8f6f4 takes a scale byte for
// each row of its operands, and its 128 values of k are one block.
#include <algorithm>

#include "mm.h"

namespace e2v2 {
namespace {

// The side of the tiles: 256 where they fill the 256 CUs (8192 x 8192 x 2048: 129 us, with tiles of 128 150) and, with
// experts, where those have rows for several and k is not short (64 experts of 512 rows, 2048 x 1408: 160 and 144; 16 of
// 2048 rows 134 and 121; 64 of 512 rows, 2048 x 4096: 350 and 358); 64 where not even those of 128 fill them (500 x 1000 x
// 1000: 7.9, and 9.8 with tiles of 128).
int tile_side(int64_t m, int64_t n, int64_t k, int groups) {
  auto tiles = [&](int64_t t) { return (m / t + (groups < m ? groups : m)) * ((n + t - 1) / t); };
  if (tiles(256) >= 200 && (groups > 1 ? k >= 2048 && m / groups >= 1024 : m >= 192)) return 256;
  return tiles(128) >= 256 ? 128 : 64;
}

// Parts of k, where the tiles are few and k is long (1024 x 1024 x 16384: 39 us, uncut 63; 128 x 1024 x 65536: 32 and 236;
// 500 x 1000 x 4096: 17 and 19; 256 x 4096 x 4096: 21 and 19).  The rule does not know whether rows start on 16 bytes: where
// they do not, calls that would have taken the pass over few rows walk k in tiles of 128, uncut (64 x 64 x 8191 packed 82 us,
// 65 rows, in parts, 21, 64 x 64 x 8192 10; 1 x 4096 x 4095 packed 52, 1 x 4096 x 4096 6).
int splits_of(int64_t m, int64_t n, int64_t k) {
  if (thin_rows(m, n, k, 1)) return 1;
  const int64_t t = tile_side(m, n, k, 1) == 256 ? 256 : 128, tiles = ((m + t - 1) / t) * ((n + t - 1) / t);
  const int64_t steps = (k + 127) / 128;
  if (tiles >= 192 || steps < 16) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>({512 / tiles, steps / 8, 16}));
}

template <int kGroup, bool kStaged>
void run8(const MmArgs& P, hipStream_t s) {
  const int side = tile_side(P.m, P.n, P.k, P.groups);
  if constexpr (!kStaged) {
    if (P.splits == 1 && thin_rows(P.m, P.n, P.k, P.groups)) return launch_thin<kE4m3, kGroup>(P, s);
    if (side == 256) return launch_mm<kE4m3, false, false, 256, 256, 2, 4, kGroup, false>(P, s);
    if (side == 64 && P.splits == 1) return launch_mm<kE4m3, false, false, 64, 64, 2, 1, kGroup, false>(P, s);
  }
  launch_mm<kE4m3, false, false, 128, 128, 2, 2, kGroup, kStaged>(P, s);
}

}  // namespace
}  // namespace e2v2

using namespace e2v2;

E2V2_API int64_t e2v2_product8_workspace(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const int splits = splits_of(m, n, k);
  return splits > 1 ? splits * m * n * 4 : 0;
}

E2V2_API int e2v2_product8(const e2v2_product8_args* a, float* ws, int64_t ws_bytes, hipStream_t s) {
  E2V2_REQUIRE(a, "product8: null arguments");
  E2V2_REQUIRE(a->m >= 0 && a->n >= 0 && a->k >= 0 && a->m <= INT32_MAX / 2 && a->n <= INT32_MAX / 2 &&
                   a->k <= INT32_MAX / 2, "product8: %lld x %lld x %lld", (long long)a->m, (long long)a->n, (long long)a->k);
  E2V2_REQUIRE(a->out_type >= E2V2_F32 && a->out_type <= E2V2_F16, "product8: output type %d", a->out_type);
  E2V2_REQUIRE(!a->offsets || a->groups > 0, "product8: %d experts", a->groups);
  if (a->m == 0 || a->n == 0) return 0;
  E2V2_REQUIRE(a->a && a->b && a->sa && a->sb && a->y, "product8: null operand");
  E2V2_REQUIRE(a->lda >= a->k && a->ldb >= a->k && a->lda <= kMaxPitch && a->ldb <= kMaxPitch && a->ldy >= a->n,
               "product8: rows %lld, %lld and %lld apart", (long long)a->lda, (long long)a->ldb, (long long)a->ldy);
  E2V2_REQUIRE((uintptr_t)a->y % (a->out_type == E2V2_F32 ? 4 : 2) == 0 && (uintptr_t)a->offsets % 4 == 0 &&
                   (uintptr_t)ws % 16 == 0, "product8: misaligned operand");
  const int64_t nb = (a->k + 127) / 128, sb_each = a->b_tiles ? (a->n + 127) / 128 : a->n;
  auto fits = [](int64_t rows, int64_t ld, int64_t blocks, int64_t step) {
    return ld >= 0 && step >= 0 && (rows - 1) * ld + (blocks - 1) * step < INT32_MAX / 2;
  };
  E2V2_REQUIRE(fits(std::min<int64_t>(a->m, 256), a->sa_ld, nb, a->sa_k) &&
                   fits(std::min<int64_t>(sb_each, 256), a->sb_ld, nb, a->sb_k),
               "product8: scales %lld and %lld apart, %lld and %lld", (long long)a->sa_ld, (long long)a->sa_k,
               (long long)a->sb_ld, (long long)a->sb_k);
  const bool grouped = a->offsets != nullptr;
  MmArgs P{};
  P.a = static_cast<const uint8_t*>(a->a);
  P.b = static_cast<const uint8_t*>(a->b);
  P.sa = a->sa;
  P.sb = a->sb;
  P.y = a->y;
  P.part = ws;
  P.offsets = a->offsets;
  P.lda = a->lda;
  P.ldb = a->ldb;
  P.b_group = a->b_group;
  P.sb_group = a->sb_group;
  P.ldy = a->ldy;
  P.sa_ld = a->sa_ld;
  P.sa_k = a->sa_k;
  P.sb_ld = a->sb_ld;
  P.sb_k = a->sb_k;
  P.m = (int)a->m;
  P.n = (int)a->n;
  P.k = (int)a->k;
  P.groups = grouped ? a->groups : 1;
  P.sb_rows = a->b_tiles ? 128 : 1;
  P.out_type = a->out_type;
  P.fill = a->fill;
  const bool staged = ((uintptr_t)a->a | (uintptr_t)a->b | (uintptr_t)a->lda | (uintptr_t)a->ldb |
                       (uintptr_t)(grouped ? a->b_group : 0)) % 16 != 0;
  P.splits = grouped ? 1 : splits_of(a->m, a->n, a->k);
  E2V2_REQUIRE(P.splits == 1 || (ws && ws_bytes >= e2v2_product8_workspace(a->m, a->n, a->k)),
               "product8: workspace of %lld bytes", (long long)ws_bytes);
  const int64_t tiles = (a->m / 16 + P.groups) * ((a->n + 15) / 16);
  E2V2_REQUIRE(tiles < INT32_MAX / 2, "product8: %lld tiles", (long long)tiles);
  if (grouped) staged ? run8<kRows, true>(P, s) : run8<kRows, false>(P, s);
  else staged ? run8<kDense, true>(P, s) : run8<kDense, false>(P, s);
  E2V2_LAUNCHED("k_mm");
  if (P.splits > 1) {
    launch_mm_sum(P, P.m, s);
    E2V2_LAUNCHED("k_mm_sum");
  }
  return 0;
}
