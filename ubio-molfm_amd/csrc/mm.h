// Tiled matrix products on MFMA: y[i][j] = sum_k a(i, k) b(j, k), for rows of 8-bit floats with block scales (fp8.hip) and
// for products grouped by expert (experts.hip), in fp32, bf16, fp16 or e4m3.
//
// Layouts.  Every operand is a matrix whose rows are consecutive.  "Inner": the reduction k runs along a row; "outer":
// rows are values of k (the weight in the product of the rows' gradient, both operands in the weight's).  A workgroup
// computes a BM x BN tile and walks k in steps of 128 bytes of an inner row (64 values of 16 bits, 32 of fp32, 128 of
// e4m3); both operands' tiles of a step lie in LDS, two steps' worth, filled by loads that write LDS themselves.
//   inner tile: [rows][128 bytes], 16-byte piece c of row r at place c ^ swizzle(r)
//   outer tile: [values of k][BM or BN elements], likewise; 16-bit operands are read from it by the transposing LDS read
// A 16-byte piece of an operand lies in one lane of a matrix instruction, so all types share the reads of inner tiles.
//
// The N side (b) is the matrix instruction's first operand and its rows are dealt so that a lane ends up with 4 FN
// consecutive columns of one row of y: lane (g, i) of fragment f takes row 4 FN (i / 4) + 4 f + i % 4.
//
// fp32 operands are split in registers into three bf16 pieces (x0 = bf16(x), x1 = bf16(x - x0), x2 = bf16(x - x0 - x1);
// the split is exact) and a product is the six piece products of order <= 2: fp32 accuracy at a sixth of the bf16 rate,
// 2.6 times that of the fp32 matrix instructions.  Accumulation is fp32 throughout; y is rounded once.  e4m3 products are added
// by eights before that, on a grid of 2^-13 of the largest of the eight: the matrix unit's own step, at twice the rate of
// any other; it adds about 2^-15 of the result's size (rms), where the operands' codes are 2^-5 off.
//
// Groups.  kRows: rows offsets[e] .. offsets[e + 1] of a meet matrix e of b; the tiles of all experts form one list, and
// each workgroup finds its own from the offsets on the GPU, so that the host never waits for them.  kRed: the reduction
// runs over the rows of expert e and there is a y for each.  Offsets are clamped to the rows there are.
#pragma once
#include <type_traits>

#include "common.h"
#include "../../include/e2v2.h"

namespace e2v2 {

enum : int { kBf16 = 0, kF16 = 1, kF32 = 2, kE4m3 = 3 };         // operand types
enum : int { kDense = 0, kRows = 1, kRed = 2 };

struct MmArgs {
  const uint8_t* a; const uint8_t* b; const uint8_t* sa; const uint8_t* sb;
  void* y; float* part;            // part: fp32 sums of each split, [splits][groups][m][n], if splits > 1
  const int* offsets;              // [groups + 1]
  int64_t lda, ldb;                // bytes from row to row
  int64_t b_group, sb_group;       // bytes from expert to expert
  int64_t ldy;                     // elements from row to row
  int64_t sa_bytes, sb_bytes;      // of all row scales of a and of b
  int m, n, k;                     // kRows: m = all rows of a; kRed: k = all rows
  int groups, tiles_m, tiles_n, splits, sb_rows, out_type;
  int fill;                        // kRows: rows of no expert become zeros
};

namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) uint8_t lds8;

constexpr int kStepBytes = 128;

constexpr int elem_size(int t) { return t == kF32 ? 4 : t == kE4m3 ? 1 : 2; }
constexpr int log2c(int v) { return v <= 1 ? 0 : 1 + log2c(v / 2); }

// Where piece c of row r of a tile lies.  kFrag: fragments whose rows are dealt over 4 kFrag consecutive ones (N side);
// 0: a fragment is 16 consecutive rows (M side).  The 16 rows (inner) or 8 to 16 pieces (outer) that a wavefront reads at
// once come to lie in different banks of LDS's 64.
template <int kT, bool kOuter, int kFrag, int kPieces>
__device__ __forceinline__ int swizzle(int r) {
  if constexpr (!kOuter) {
    if constexpr (kFrag <= 1) return (r >> 1) & 7;
    else return ((r >> 1) & 1) | (((r >> log2c(4 * kFrag)) & 3) << 1);
  } else if constexpr (kT == kF32) {
    if constexpr (kFrag == 0) return ((r >> 2) & 3) << 2 & (kPieces - 1);
    else return (r >> 2) & 3;
  } else {
    if constexpr (kFrag == 0) return ((r & 3) | ((r >> 3) & 1) << 2) << 1 & (kPieces - 1);
    else return ((r & 1) | ((r >> 1) & 1) << 3) & (kPieces - 1);
  }
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t u = (uint64_t)p;
  return (const uint8_t*)((uint64_t)(uint32_t)uniform((int)u) | (uint64_t)(uint32_t)uniform((int)(u >> 32)) << 32);
}

// Loads of one operand's tiles: R rows of y's side, NT threads.  A buffer's range covers exactly what the tile may read;
// pieces out of it read as zero.  kStaged: rows on any byte boundary (16-byte pieces are put together from aligned
// dwords) or ends inside a piece, through registers.
template <int kT, bool kOuter, int kFrag, int R, int NT, bool kStaged>
struct TileLoad {
  static constexpr int es = elem_size(kT), kK = kStepBytes / es, kPieces = kOuter ? R * es / 16 : 8;
  static constexpr int kRounds = R * 8 / NT, kBytes = R * kStepBytes;
  static constexpr unsigned kNowhere = 0xf0000000u;
  int off[kRounds];
  intx4 hold[kStaged ? kRounds : 1];
  const uint8_t* base;
  int64_t ld;
  int width;                       // inner: bytes of k; outer: bytes of the tile's columns that there are
  int rows;                        // inner: rows there are; outer: values of k there are

  // p: the tile's first element; inner: rows below it and k values; outer: columns from it on and k values.
  __device__ __forceinline__ void start(const uint8_t* p, int64_t ld_, int extent, int k) {
    base = p;
    ld = ld_;
    if constexpr (kOuter) { width = min(extent, R) * es; rows = k; }
    else { width = k * es; rows = min(extent, R); }
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
      const int q = j * NT + threadIdx.x, r = q / kPieces, c = (q % kPieces) ^ swizzle<kT, kOuter, kFrag, kPieces>(r);
      off[j] = (int)(r * ld + c * 16);
    }
  }

  // The address and bytes of step t's part: inner rows are read from their own start.
  __device__ __forceinline__ intx4 range(int t, int& skew) const {
    const uint8_t* p = base;
    int64_t bytes;
    if constexpr (kOuter) {
      const int left = min(rows - t * kK, kK);
      p += (int64_t)t * kK * ld;
      bytes = left > 0 ? (left - 1) * ld + width : 0;
    } else {
      bytes = rows > 0 ? (rows - 1) * ld + width : 0;
    }
    skew = 0;
    if constexpr (kStaged) {
      skew = (int)((uint64_t)p & 3);
      p -= skew;
      bytes = (bytes + skew + 3) & ~(int64_t)3;
    } else {
      bytes = (bytes + 15) & ~(int64_t)15;         // whole pieces: what lies behind the end is cleared or not used
    }
    p = uniform(p);
    return intx4{(int)(uint64_t)p, (int)((uint64_t)p >> 32) & 0xffff, uniform((int)bytes), 0x00020000};
  }

  // Sends step t's pieces on their way: into LDS at `to`, or (kStaged) into registers.
  __device__ __forceinline__ void issue(int t, lds8* to) {
    int skew;
    const intx4 srd = range(t, skew);
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
        (void*)((uint64_t)(uint32_t)srd[0] | (uint64_t)(uint32_t)srd[1] << 32), 0, srd[2], srd[3]);
    const bool tail = !kOuter && (t + 1) * kStepBytes > width;
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
      unsigned o = (unsigned)off[j];
      if constexpr (!kOuter) o += t * kStepBytes;
      if constexpr (!kStaged) {
        if (tail) {
          const int q = j * NT + threadIdx.x, r = q / kPieces, c = (q % kPieces) ^ swizzle<kT, kOuter, kFrag, kPieces>(r);
          if (t * kStepBytes + c * 16 >= width) o = kNowhere;
        }
        const int at = uniform(j * NT * 16 + (int)(threadIdx.x & ~63u) * 16);
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                     ::"s"((int)(uintptr_t)(to + at)), "v"(o), "s"(srd) : "memory");
      } else {
        o += skew;
        const intx4 lo = __builtin_amdgcn_raw_buffer_load_b128(rsrc, o & ~3u, 0, 0);
        const int hi = __builtin_amdgcn_raw_buffer_load_b32(rsrc, (o & ~3u) + 16, 0, 0);
        intx4 v;
        v[0] = __builtin_amdgcn_alignbyte(lo[1], lo[0], o & 3);
        v[1] = __builtin_amdgcn_alignbyte(lo[2], lo[1], o & 3);
        v[2] = __builtin_amdgcn_alignbyte(lo[3], lo[2], o & 3);
        v[3] = __builtin_amdgcn_alignbyte(hi, lo[3], o & 3);
        const int q = j * NT + threadIdx.x, r = q / kPieces, c = (q % kPieces) ^ swizzle<kT, kOuter, kFrag, kPieces>(r);
        // bytes of the piece that belong to the operand (values of k past the end are zeros)
        int have = 16;
        if constexpr (kOuter) have = t * kK + r < rows ? 16 : 0;
        else have = min(max(width - (t * kStepBytes + c * 16), 0), 16);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int h = have - 4 * d;
          v[d] = h >= 4 ? v[d] : h <= 0 ? 0 : v[d] & (int)((1u << (8 * h)) - 1u);
        }
        hold[j] = v;
      }
    }
  }

  // The bytes of step t's tile that lie behind the end of k in a piece that k ends in.
  __device__ __forceinline__ void clear_tail(int t, lds8* tile) const {
    if constexpr (!kOuter && !kStaged) {
      const int at = width - t * kStepBytes, r = threadIdx.x;
      if (r < R) {
        auto* p = reinterpret_cast<__attribute__((address_space(3))) uint32_t*>(
            tile + r * kStepBytes + (((at >> 4) ^ swizzle<kT, kOuter, kFrag, kPieces>(r)) << 4));
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int h = (at & 15) - 4 * d;
          if (h < 4) p[d] = h <= 0 ? 0u : p[d] & ((1u << (8 * h)) - 1u);
        }
      }
    }
  }

  __device__ __forceinline__ void put(lds8* to) const {
    if constexpr (kStaged) {
#pragma unroll
      for (int j = 0; j < kRounds; ++j)
        *reinterpret_cast<__attribute__((address_space(3))) intx4*>(to + (j * NT + threadIdx.x) * 16) = hold[j];
    }
  }
};

// A lane's part of a fragment of 16 rows of one step: two 16-byte pieces, values of k of the two halves of the step.
template <int kT, bool kOuter, int kFrag, int R>
__device__ __forceinline__ void read_frag(const lds8* tile, int first, int f, intx4 (&v)[2]) {
  const int i = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  constexpr int es = elem_size(kT), kPieces = kOuter ? R * es / 16 : 8;
  typedef __attribute__((address_space(3))) const intx4 piece;
  if constexpr (!kOuter) {
    const int r = first + (kFrag > 0 ? (i >> 2) * 4 * kFrag + f * 4 + (i & 3) : f * 16 + i);
    const int z = swizzle<kT, kOuter, kFrag, kPieces>(r);
    const lds8* row = tile + r * kStepBytes;
    v[0] = *reinterpret_cast<piece*>(row + ((g ^ z) << 4));
    v[1] = *reinterpret_cast<piece*>(row + (((g + 4) ^ z) << 4));
  } else if constexpr (kT == kF32) {
    const int col = first + (kFrag > 0 ? (i >> 2) * 4 * kFrag + f * 4 + (i & 3) : f * 16 + i);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = h * 16 + g * 4 + e;
        const int at = k * R * 4 + (((col >> 2) ^ swizzle<kT, kOuter, kFrag, kPieces>(k)) << 4) + (col & 3) * 4;
        v[h][e] = *reinterpret_cast<__attribute__((address_space(3))) const int*>(tile + at);
      }
  } else {
    // the transposing read: 16 lanes give the addresses of 4 values of k times 16 columns, lane j those of value j / 4
    // and columns 4 (j % 4) .. + 3, and lane i gets column i's four values
    const int col = first + (kFrag > 0 ? (i & 3) * 4 * kFrag + f * 4 : f * 16 + (i & 3) * 4);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      shortx4 t[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int k = h * 32 + g * 8 + e * 4 + (i >> 2);
        const int at = k * R * 2 + (((col >> 3) ^ swizzle<kT, kOuter, kFrag, kPieces>(k)) << 4) + (col & 7) * 2;
        t[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4*)(tile + at));
      }
      typedef short shortx8 __attribute__((ext_vector_type(8)));
      v[h] = __builtin_bit_cast(intx4, (shortx8)__builtin_shufflevector(t[0], t[1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
}

// A fragment as the matrix instructions take it.
template <int kT>
struct Frag {
  intx4 v[2];
  __device__ __forceinline__ void take(const intx4 (&u)[2]) { v[0] = u[0], v[1] = u[1]; }
};
template <>
struct Frag<kF32> {
  bf16x8 p[3];
  __device__ __forceinline__ void take(const intx4 (&u)[2]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = __builtin_bit_cast(float, (int)u[e >> 2][e & 3]);
      const __bf16 x0 = (__bf16)x;
      const float r1 = x - (float)x0;
      const __bf16 x1 = (__bf16)r1;
      p[0][e] = x0;
      p[1][e] = x1;
      p[2][e] = (__bf16)(r1 - (float)x1);
    }
  }
};

template <int kT>
__device__ __forceinline__ floatx4 multiply(const Frag<kT>& b, const Frag<kT>& a, floatx4 c, int sb, int sa) {
  if constexpr (kT == kE4m3) {
    const intx8 x = __builtin_shufflevector(b.v[0], b.v[1], 0, 1, 2, 3, 4, 5, 6, 7);
    const intx8 y = __builtin_shufflevector(a.v[0], a.v[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 0, 0, 0, sb, 0, sa);
  } else if constexpr (kT == kF32) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.p[2], a.p[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.p[1], a.p[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.p[0], a.p[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.p[1], a.p[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.p[0], a.p[1], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.p[0], a.p[0], c, 0, 0, 0);
  } else if constexpr (kT == kBf16) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b.v[0]), __builtin_bit_cast(bf16x8, a.v[0]), c,
                                                0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b.v[1]), __builtin_bit_cast(bf16x8, a.v[1]),
                                                   c, 0, 0, 0);
  } else {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b.v[0]), __builtin_bit_cast(f16x8, a.v[0]), c,
                                               0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b.v[1]), __builtin_bit_cast(f16x8, a.v[1]), c,
                                                  0, 0, 0);
  }
}

// Four scale bytes from byte `at` on of a table of `bytes`; bytes past its end are not read.
__device__ __forceinline__ uint32_t scales4(const uint8_t* p, int64_t at, int64_t bytes) {
  typedef uint32_t any __attribute__((aligned(1)));
  if (bytes >= 4) {
    const int64_t from = min(at, bytes - 4);
    return *reinterpret_cast<const any*>(p + from) >> (8 * (int)min(at - from, (int64_t)3));
  }
  uint32_t v = 0;
  for (int e = 0; e < 3; ++e)
    if (at + e < bytes) v |= (uint32_t)p[at + e] << (8 * e);
  return v;
}

// Expert e's rows; e = groups and groups + 1: those before the first expert's and behind the last one's.
__device__ __forceinline__ void expert_rows(const MmArgs& P, int total, int e, int& s, int& t) {
  const int E = P.groups;
  auto clamp = [](int v, int lo, int hi) { return min(max(v, lo), hi); };
  if (e < E) {
    s = clamp(P.offsets[e], 0, total);
    t = clamp(P.offsets[e + 1], s, total);
  } else if (e == E) {
    s = 0;
    t = P.fill ? clamp(P.offsets[0], 0, total) : 0;
  } else {
    s = clamp(P.offsets[E], clamp(P.offsets[E - 1], 0, total), total);
    t = P.fill && e == E + 1 ? total : s;
  }
}

struct Tile {
  int e, row0, rows, mt, nt;       // rows row0 .. row0 + rows belong to the tile's expert from the tile's first on
  bool any, zero;
};

__device__ __forceinline__ int of_xcd(int total, bool& any) {
  const int per = (total + kXcd - 1) / kXcd, at = (int)blockIdx.x / kXcd;
  const int id = (int)blockIdx.x % kXcd * per + at;
  any = at < per && id < total;
  return id;
}

// The workgroup's tile.  Every XCD takes a consecutive part of the list, so that tiles that share rows or columns share
// its L2.
template <int kGroup, int BM>
__device__ __forceinline__ Tile find_tile(const MmArgs& P) {
  Tile T;
  T.zero = false;
  T.e = 0;
  if constexpr (kGroup == kRows) {
    const int lane = threadIdx.x & 63, all = P.groups + 2;
    int total = 0, s, t, count = 0, incl = 0;
    for (int e0 = 0; e0 < all; e0 += 64) {
      if (e0 + lane < all) expert_rows(P, P.m, e0 + lane, s, t);
      else s = t = 0;
      count = (t - s + BM - 1) / BM;
      incl = count;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(incl, o, 64);
        if (lane >= o) incl += v;
      }
      incl += total;
      total = __shfl(incl, 63, 64);
    }
    const int id = of_xcd(total * P.tiles_n, T.any);
    if (!T.any) return T;
    const int mt = id / P.tiles_n;
    T.nt = id - mt * P.tiles_n;
    int before = 0;
    for (int e0 = 0; e0 < all; e0 += 64) {
      if (all > 64) {                              // else the only part's values are still there
        if (e0 + lane < all) expert_rows(P, P.m, e0 + lane, s, t);
        else s = t = 0;
        count = (t - s + BM - 1) / BM;
        incl = count;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int v = __shfl_up(incl, o, 64);
          if (lane >= o) incl += v;
        }
        incl += before;
      }
      const uint64_t hit = __ballot(incl > mt);
      if (hit) {
        const int h = __builtin_ctzll(hit);
        T.e = uniform(e0 + h);
        T.mt = uniform(mt - (__shfl(incl, h, 64) - __shfl(count, h, 64)));
        T.row0 = uniform(__shfl(s, h, 64) + T.mt * BM);
        T.rows = uniform(__shfl(t, h, 64) - T.row0);
        break;
      }
      before = __shfl(incl, 63, 64);
    }
    T.zero = T.e >= P.groups;
    return T;
  } else {
    const int each = P.tiles_m * P.tiles_n;
    int id = of_xcd(each * (kGroup == kRed ? P.groups : 1), T.any);
    if (!T.any) return T;
    if constexpr (kGroup == kRed) {
      T.e = id / each;
      id -= T.e * each;
    }
    // eight rows of tiles at a time, column by column: the 32 tiles that an XCD works on at once read 8 and 4 operands
    const int block = 8 * P.tiles_n, b = id / block, in = id - b * block, high = min(P.tiles_m - b * 8, 8);
    T.nt = in / high;
    T.mt = b * 8 + in - T.nt * high;
    T.row0 = T.mt * BM;
    T.rows = P.m - T.row0;
    return T;
  }
}

// kN values of a row of y from column c on, n columns in all.
template <typename T, int kN>
__device__ __forceinline__ void put_row(T* row, int c, int n, bool aligned, const float (&v)[kN]) {
  constexpr int V = 16 / sizeof(T) < kN ? 16 / sizeof(T) : kN;
  typedef T vec __attribute__((ext_vector_type(V)));
  if (aligned && c + kN <= n) {
#pragma unroll
    for (int k = 0; k < kN; k += V) {
      vec o;
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = (T)v[k + e];
      *reinterpret_cast<vec*>(row + c + k) = o;
    }
  } else {
#pragma unroll
    for (int e = 0; e < kN; ++e)
      if (c + e < n) row[c + e] = (T)v[e];
  }
}

template <int kN>
__device__ __forceinline__ void put(void* y, int64_t at, int c, int n, int64_t ld, int type, const float (&v)[kN]) {
  const int size = type == E2V2_F32 ? 4 : 2;
  const bool aligned = (((uint64_t)y | (uint64_t)(ld * size)) & 15) == 0;
  if (type == E2V2_F32) put_row<float, kN>(static_cast<float*>(y) + at, c, n, aligned, v);
  else if (type == E2V2_BF16) put_row<__bf16, kN>(static_cast<__bf16*>(y) + at, c, n, aligned, v);
  else put_row<_Float16, kN>(static_cast<_Float16*>(y) + at, c, n, aligned, v);
}

// kAO, kBO: outer layout of a, b.  WM x WN wavefronts.
template <int kT, bool kAO, bool kBO, int BM, int BN, int WM, int WN, int kGroup, bool kStaged>
__global__ __launch_bounds__(WM * WN * 64) void k_mm(MmArgs P) {
  constexpr int NT = WM * WN * 64, FM = BM / WM / 16, FN = BN / WN / 16, es = elem_size(kT), kK = kStepBytes / es;
  __shared__ __attribute__((aligned(1024))) uint8_t mem[2][(BM + BN) * kStepBytes];
  const Tile T = find_tile<kGroup, BM>(P);
  if (!T.any) return;
  const int wave = uniform((int)threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  const int i = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  const int n0 = T.nt * BN;

  // the reduction's part: of all of k, or of the expert's rows
  int k0 = 0, k1 = P.k;
  if constexpr (kGroup == kRed) expert_rows(P, P.k, T.e, k0, k1);
  if (P.splits > 1) {
    const int steps = (k1 - k0 + kK - 1) / kK, each = (steps + P.splits - 1) / P.splits * kK;
    k1 = min(k1, k0 + ((int)blockIdx.y + 1) * each);
    k0 = min(k0 + (int)blockIdx.y * each, k1);
  }
  const int steps = T.zero ? 0 : (k1 - k0 + kK - 1) / kK;

  TileLoad<kT, kAO, 0, BM, NT, kStaged> la;
  TileLoad<kT, kBO, FN, BN, NT, kStaged> lb;
  {
    const uint8_t* pb = P.b + (kGroup == kRows ? (int64_t)T.e * P.b_group : 0);
    if constexpr (kAO) la.start(P.a + (int64_t)k0 * P.lda + (int64_t)T.row0 * es, P.lda, T.rows, k1 - k0);
    else la.start(P.a + (int64_t)T.row0 * P.lda + (int64_t)k0 * es, P.lda, T.rows, k1 - k0);
    if constexpr (kBO) lb.start(pb + (int64_t)k0 * P.ldb + (int64_t)n0 * es, P.ldb, P.n - n0, k1 - k0);
    else lb.start(pb + (int64_t)n0 * P.ldb + (int64_t)k0 * es, P.ldb, P.n - n0, k1 - k0);
  }

  floatx4 acc[FM][FN];
#pragma unroll
  for (int f = 0; f < FM; ++f)
#pragma unroll
    for (int h = 0; h < FN; ++h) acc[f][h] = floatx4{0.f, 0.f, 0.f, 0.f};

  // scale bytes of four steps, and of the next four
  constexpr int SA = kT == kE4m3 ? FM : 1, SB = kT == kE4m3 ? FN : 1;
  uint32_t sa[SA], sb[SB], sa_next[SA], sb_next[SB];
  const int nb = (P.k + 127) / 128, kb0 = k0 / 128;
  auto load_scales = [&](int t) {
    if constexpr (kT == kE4m3) {
#pragma unroll
      for (int f = 0; f < FM; ++f) {
        const int64_t r = T.row0 + min(wm * FM * 16 + f * 16 + i, T.rows - 1);
        sa_next[f] = scales4(P.sa, r * nb + kb0 + t, P.sa_bytes);
      }
      const uint8_t* p = P.sb + (kGroup == kRows ? (int64_t)T.e * P.sb_group : 0);
#pragma unroll
      for (int h = 0; h < FN; ++h) {
        const int r = min(n0 + wn * FN * 16 + (i >> 2) * 4 * FN + h * 4 + (i & 3), P.n - 1);
        sb_next[h] = scales4(p, (int64_t)(P.sb_rows > 1 ? r / 128 : r) * nb + kb0 + t, P.sb_bytes);
      }
    }
  };

  auto buf = [&](int t) { return (lds8*)mem[t & 1]; };
  auto fetch = [&](int t) {
    la.issue(t, buf(t));
    lb.issue(t, buf(t) + BM * kStepBytes);
  };
  if (steps > 0) {
    load_scales(0);
    fetch(0);
  }
  for (int t = 0; t < steps; ++t) {
    if constexpr (kStaged) {
      la.put(buf(t));
      lb.put(buf(t) + BM * kStepBytes);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if constexpr (!kStaged && !(kAO && kBO)) {
      if (t + 1 == steps && ((k1 - k0) * es & 15)) {
        la.clear_tail(t, buf(t));
        lb.clear_tail(t, buf(t) + BM * kStepBytes);
        __syncthreads();
      }
    }
    if (t + 1 < steps) fetch(t + 1);
    if constexpr (kT == kE4m3) {
      if ((t & 3) == 0) {
#pragma unroll
        for (int f = 0; f < FM; ++f) sa[f] = sa_next[f];
#pragma unroll
        for (int h = 0; h < FN; ++h) sb[h] = sb_next[h];
        if (t + 4 < steps) load_scales(t + 4);
      }
    }
    const lds8* ta = buf(t);
    const lds8* tb = ta + BM * kStepBytes;
    Frag<kT> fb[FN];
#pragma unroll
    for (int h = 0; h < FN; ++h) {
      intx4 u[2];
      read_frag<kT, kBO, FN, BN>(tb, wn * FN * 16, h, u);
      fb[h].take(u);
    }
#pragma unroll
    for (int f = 0; f < FM; ++f) {
      intx4 u[2];
      Frag<kT> fa;
      read_frag<kT, kAO, 0, BM>(ta, wm * FM * 16, f, u);
      fa.take(u);
#pragma unroll
      for (int h = 0; h < FN; ++h) {
        if constexpr (kT == kE4m3)
          acc[f][h] = multiply<kT>(fb[h], fa, acc[f][h], (int)(sb[h] >> (8 * (t & 3))), (int)(sa[f] >> (8 * (t & 3))));
        else acc[f][h] = multiply<kT>(fb[h], fa, acc[f][h], 0, 0);
      }
    }
  }

  // lane (g, i) holds row i of each fragment and 4 FN columns of it
  const int c = n0 + wn * FN * 16 + g * 4 * FN;
#pragma unroll
  for (int f = 0; f < FM; ++f) {
    const int r = wm * FM * 16 + f * 16 + i;
    if (r >= T.rows) continue;
    float v[4 * FN];
#pragma unroll
    for (int h = 0; h < FN; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[h * 4 + e] = acc[f][h][e];
    const int64_t plane = kGroup == kRed ? T.e : 0;
    if (P.splits > 1) {
      const int64_t at = ((((int64_t)blockIdx.y * (kGroup == kRed ? P.groups : 1) + plane) * P.m) + T.row0 + r) * P.n;
      put<4 * FN>(P.part, at, c, P.n, P.n, E2V2_F32, v);
    } else {
      put<4 * FN>(P.y, (plane * P.m + T.row0 + r) * P.ldy, c, P.n, P.ldy, P.out_type, v);
    }
  }
}

// y = the sum of the splits' parts, in order, rounded once.
__global__ __launch_bounds__(256) void k_mm_sum(const float* part, int splits, int64_t rows, int n, void* y, int64_t ldy,
                                                int type) {
  const int64_t all = rows * n, stride = (int64_t)gridDim.x * 256;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < all; at += stride) {
    float s = 0.f;
    for (int k = 0; k < splits; ++k) s += part[k * all + at];
    const int64_t to = ldy == n ? at : at / n * ldy + at % n;
    if (type == E2V2_F32) static_cast<float*>(y)[to] = s;
    else if (type == E2V2_BF16) static_cast<__bf16*>(y)[to] = (__bf16)s;
    else static_cast<_Float16*>(y)[to] = (_Float16)s;
  }
}

template <int kT, bool kAO, bool kBO, int BM, int BN, int WM, int WN, int kGroup, bool kStaged>
void launch_mm(MmArgs P, hipStream_t s) {
  P.tiles_n = (P.n + BN - 1) / BN;
  P.tiles_m = (P.m + BM - 1) / BM;
  int64_t tiles;
  if constexpr (kGroup == kRows) tiles = (int64_t)(P.m / BM + P.groups + 2) * P.tiles_n;
  else tiles = (int64_t)P.tiles_m * P.tiles_n * (kGroup == kRed ? P.groups : 1);
  tiles = (tiles + kXcd - 1) / kXcd * kXcd;
  hipLaunchKernelGGL((k_mm<kT, kAO, kBO, BM, BN, WM, WN, kGroup, kStaged>), dim3((unsigned)tiles, (unsigned)P.splits),
                     dim3(WM * WN * 64), 0, s, P);
}

inline void launch_mm_sum(const MmArgs& P, int64_t rows, hipStream_t s) {
  const int64_t blocks = (rows * P.n + 255) / 256;
  hipLaunchKernelGGL(k_mm_sum, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, P.part, P.splits, rows,
                     P.n, P.y, P.ldy, P.out_type);
}

}  // namespace
}  // namespace e2v2
