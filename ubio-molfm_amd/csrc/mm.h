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
// The N side (b) is the matrix instruction's first operand and its rows are dealt so that a lane ends up with eight
// consecutive columns of a row of y for each two fragments, and the four lanes of that row with 32: lane (g, i) of
// fragment f takes row 32 (f / 2) + 8 (i / 4) + 4 (f % 2) + i % 4.
//
// fp32 operands are split in registers into three bf16 pieces (x0 = x cut to bf16, x1 = bf16(x - x0), x2 = x - x0 - x1: the
// split is exact) and a product is the six piece products of order <= 2.  What is left out is at most 2^-22 of each product
// (|x1| < 2^-7 |x|, |x2| <= 2^-16 |x|) and of either sign: fp32 accuracy at a sixth of the bf16 rate, 2.6 times that of the
// fp32 matrix instructions.  Accumulation is fp32 throughout; y is rounded once.  e4m3 products are added
// by eights before that, on a grid of 2^-13 of the largest of the eight: the matrix unit's own step, at twice the rate of
// any other; it adds 2^-16 to 2^-13 of the result's size (rms), where codes are up to 2^-4 of theirs off.
//
// Groups.  kRows: rows offsets[e] .. offsets[e + 1] of a meet matrix e of b; the tiles of all experts form one list, and
// each workgroup finds its own from the offsets on the GPU, so that the host never waits for them.  kRed: the reduction
// runs over the rows of expert e and there is a y for each.  Offsets are clamped to the rows there are.
#pragma once
#include <algorithm>
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
  int64_t sa_ld, sa_k, sb_ld, sb_k;   // bytes from row to row and from block to block of the scales
  int m, n, k;                     // kRows: m = all rows of a; kRed: k = all rows
  int groups, tiles_m, tiles_n, splits, sb_rows, out_type;
  int share;                       // kRed: tiles of an expert that follow one another on one XCD
  int fill;                        // kRows: rows of no expert become zeros
};

namespace {

// The kernel's arguments where they lie.  Read anew in each place that needs them: held in registers through the loop they
// pushed others out.
typedef const __attribute__((address_space(4))) MmArgs Args;
__device__ __forceinline__ Args& arguments() {
  Args* p = (Args*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
}

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) uint8_t lds8;

constexpr int kStepBytes = 128;
constexpr int64_t kMaxPitch = 1 << 22;           // bytes between rows: a tile's offsets stay below 2^30

constexpr int elem_size(int t) { return t == kF32 ? 4 : t == kE4m3 ? 1 : 2; }

// The row of a tile that lane i of fragment f takes.  kDealt: the N side's order, else 16 consecutive rows.
template <bool kDealt>
__device__ __forceinline__ int frag_row(int f, int i) {
  return kDealt ? (f >> 1) * 32 + (i >> 2) * 8 + (f & 1) * 4 + (i & 3) : f * 16 + i;
}

// Where piece c of row r of a tile lies: c ^ this.  The 16 rows (inner) or 8 to 16 pieces (outer) that a wavefront reads at
// once come to lie in different banks of LDS's 64.
template <int kT, bool kOuter, bool kDealt, int kPieces>
__device__ __forceinline__ int swizzle(int r) {
  if constexpr (!kOuter) return kDealt ? ((r >> 1) & 1) | (((r >> 3) & 3) << 1) : (r >> 1) & 7;
  else if constexpr (kT == kF32) return kDealt ? ((r >> 2) & 1) | ((r >> 3) & 1) << 3 : ((r >> 2) & 3) << 2;
  else return (kDealt ? (r & 3) << 2 : ((r & 3) | ((r >> 3) & 1) << 2) << 1) & (kPieces - 1);
}

// f(integral_constant) for 0 .. kN - 1
template <int kN, int kAt = 0, typename F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (kAt < kN) {
    f(std::integral_constant<int, kAt>{});
    each<kN, kAt + 1>(f);
  }
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t u = (uint64_t)p;
  return (const uint8_t*)((uint64_t)(uint32_t)uniform((int)u) | (uint64_t)(uint32_t)uniform((int)(u >> 32)) << 32);
}

// A load of the calling lanes' pieces of `kBytes` that writes LDS itself, at `to` + kAt onwards (uniform; lane l's at 16 l,
// single bytes as dwords at 4 l).  `step` is added to the addresses; whether it counts in the range check is left open.
template <int kBytes, int kAt>
__device__ __forceinline__ void load_to_lds(int to, unsigned off, intx4 srd, int step) {
  if constexpr (kBytes == 16)
    asm volatile("s_add_u32 m0, %0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 ::"s"(to), "v"(off), "s"(srd), "s"(step), "n"(kAt) : "memory", "scc");
  else
    asm volatile("s_add_u32 m0, %0, %4\n\ts_nop 0\n\tbuffer_load_ubyte %1, %2, %3 offen lds"
                 ::"s"(to), "v"(off), "s"(srd), "s"(step), "n"(kAt) : "memory", "scc");
}

constexpr unsigned kNowhere = 0xf0000000u;         // an offset out of every range: such pieces read as zero

// The descriptor of a buffer of these bytes.
__device__ __forceinline__ intx4 descriptor(const uint8_t* p, int bytes) {
  p = uniform(p);
  return intx4{(int)(uint64_t)p, (int)((uint64_t)p >> 32) & 0xffff, uniform(bytes), 0x00020000};
}

// Loads of one operand's tiles: R rows of y's side, NT threads.  A buffer's range covers exactly what the tile may read;
// pieces out of it read as zero.  kStaged: rows on any byte boundary (16-byte pieces are put together from aligned
// dwords), through registers.
template <int kT, bool kOuter, bool kDealt, int R, int NT, bool kStaged>
struct TileLoad {
  static constexpr int es = elem_size(kT), kK = kStepBytes / es, kPieces = kOuter ? R * es / 16 : 8;
  static constexpr int kRounds = R * 8 / NT;
  // rows from round to round; where they keep the swizzle, a thread's pieces lie at one place of their rows
  static constexpr int kStride = NT / kPieces;
  static constexpr bool kEven = kOuter ? es == 2 && kStride % 16 == 0 : kStride % 32 == 0;
  unsigned off[kEven ? 1 : kRounds];
  intx4 hold[kStaged ? kRounds : 1];
  const uint8_t* base;
  int ld;
  intx4 srd;                       // direct: of the step that is sent
  int width;                       // inner: bytes of k; outer: bytes of the tile's columns that there are
  int rows;                        // inner: rows there are; outer: values of k there are
  int step;
  unsigned dead;                   // inner: a bit for each place of the lane's pieces that lies behind the end of k

  // The thread's row and piece of it in round j.
  __device__ __forceinline__ static void piece(int j, int& r, int& c) {
    const int q = j * NT + threadIdx.x;
    r = q / kPieces;
    c = (q % kPieces) ^ swizzle<kT, kOuter, kDealt, kPieces>(r);
  }

  // p: the tile's first element; inner: rows below it and k values; outer: columns from it on and k values.
  __device__ __forceinline__ void start(const uint8_t* p, int ld_, int extent, int k) {
    base = p;
    ld = ld_;
    if constexpr (kOuter) { width = min(extent, R) * es; rows = k; }
    else { width = k * es; rows = min(extent, R); }
#pragma unroll
    for (int j = 0; j < (kEven ? 1 : kRounds); ++j) {
      int r, c;
      piece(j, r, c);
      off[j] = (unsigned)(r * ld + c * 16);
    }
    if constexpr (!kStaged) srd = descriptor(p, bytes(0));
  }

  // The bytes that step t may read: whole pieces in direct loads (what lies behind the end is cleared or not used).
  __device__ __forceinline__ int bytes(int t) const {
    int v;
    if constexpr (kOuter) {
      const int left = min(rows - t * kK, kK);
      v = left > 0 ? (left - 1) * ld + width : 0;
    } else {
      v = rows > 0 ? (rows - 1) * ld + width : 0;
    }
    return kStaged ? v : (v + 15) & ~15;
  }

  // No tile is left: what is sent reads nothing.
  __device__ __forceinline__ void stop() {
    if constexpr (!kStaged) srd[2] = 0, rows = 0, base = nullptr, width = 0;
  }

  template <int j>
  __device__ __forceinline__ unsigned place() const {
    return kEven ? off[0] + (unsigned)(j * kStride * ld) : off[kEven ? 0 : j];
  }

  // Before the rounds of step t.
  __device__ __forceinline__ void prepare(int t) {
    if constexpr (!kStaged) {
      if constexpr (kOuter) {
        srd = descriptor(base + (int64_t)t * kK * ld, bytes(t));
        step = 0;
      } else {
        step = t * kStepBytes;
        dead = 0;
        if (step + kStepBytes > width) {           // the same for all
#pragma unroll
          for (int j = 0; j < (kEven ? 1 : kRounds); ++j) {
            int r, c;
            piece(j, r, c);
            dead |= step + c * 16 >= width ? 1u << j : 0u;
          }
        }
      }
    }
  }
  // Round j of the step into LDS at `to`, the wavefront's part.
  template <int j>
  __device__ __forceinline__ void send(int to) const {
    load_to_lds<16, j * NT * 16>(to, !kOuter && (dead >> (kEven ? 0 : j) & 1) ? kNowhere : place<j>(), srd, step);
  }

  // kStaged: step t's pieces into registers.
  __device__ __forceinline__ void take(int t) {
    if constexpr (kStaged) {
      const uint8_t* p = base + (kOuter ? (int64_t)t * kK * ld : 0);
      const int skew = (int)((uint64_t)p & 3), n = bytes(t);
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)uniform(p - skew), 0,
                                                          uniform(n > 0 ? (n + skew + 3) & ~3 : 0), 0x00020000);
      each<kRounds>([&](auto j) {
        const unsigned o = place<j>() + skew + (kOuter ? 0 : t * kStepBytes);
        const intx4 lo = __builtin_amdgcn_raw_buffer_load_b128(rsrc, o & ~3u, 0, 0);
        const int hi = __builtin_amdgcn_raw_buffer_load_b32(rsrc, (o & ~3u) + 16, 0, 0);
        intx4 v;
        v[0] = __builtin_amdgcn_alignbyte(lo[1], lo[0], o & 3);
        v[1] = __builtin_amdgcn_alignbyte(lo[2], lo[1], o & 3);
        v[2] = __builtin_amdgcn_alignbyte(lo[3], lo[2], o & 3);
        v[3] = __builtin_amdgcn_alignbyte(hi, lo[3], o & 3);
        int r, c;
        piece(j, r, c);
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
      });
    }
  }

  __device__ __forceinline__ void put(lds8* to) const {
    if constexpr (kStaged) {
#pragma unroll
      for (int j = 0; j < kRounds; ++j)
        *reinterpret_cast<__attribute__((address_space(3))) intx4*>(to + (j * NT + threadIdx.x) * 16) = hold[j];
    }
  }

  // Clears the bytes of a tile's last step that lie behind the end of k, byte `at` of the step, in a piece that k ends in.
  __device__ __forceinline__ static void clear_tail(int at, lds8* tile) {
    if constexpr (!kOuter && !kStaged) {
      const int r = threadIdx.x;
      if (r < R) {
        auto* p = reinterpret_cast<__attribute__((address_space(3))) uint32_t*>(
            tile + r * kStepBytes + (((at >> 4) ^ swizzle<kT, kOuter, kDealt, kPieces>(r)) << 4));
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int h = (at & 15) - 4 * d;
          if (h < 4) p[d] = h <= 0 ? 0u : p[d] & ((1u << (8 * h)) - 1u);
        }
      }
    }
  }
};

// The scale bytes of a step, one for each row of both tiles (a tile's for all rows that it covers): a dword each in LDS,
// four steps' worth in turn.
template <int BM, int BN, int NT>
struct ScaleLoad {
  static_assert(BM + BN == NT, "a thread a row");
  static constexpr int kBytes = NT * 4;
  intx4 srd;
  unsigned off;
  int step, blocks;

  // The table's first byte of the wavefront's side, bytes between rows and blocks, rows and blocks there are, rows that share
  // a scale (1 or 128).
  __device__ __forceinline__ void start(const uint8_t* p, int64_t ld, int64_t ks, int rows, int blocks_, int each) {
    blocks = blocks_;
    const int wave = uniform((int)threadIdx.x >> 6), r = (int)threadIdx.x - (wave * 64 < BM ? 0 : BM);
    const int last = each > 1 ? (rows - 1) / 128 : rows - 1;
    srd = descriptor(p, rows > 0 && blocks > 0 ? last * (int)ld + (blocks - 1) * (int)ks + 1 : 0);
    off = (unsigned)(min(each > 1 ? r / 128 : r, last) * (int)ld);
    step = uniform((int)ks);
  }

  __device__ __forceinline__ void stop() { blocks = 0; }

  // `to`: the wavefront's part of the ring's first step.
  __device__ __forceinline__ void send(int t, int c, int to) const {
    load_to_lds<1, 0>(to + (c & 3) * kBytes, t < blocks ? off : kNowhere, srd, uniform(t < blocks ? t * step : 0));
  }
};

// A lane's part of a fragment of 16 rows of one step: two 16-byte pieces, values of k of the two halves of the step.
template <int kT, bool kOuter, bool kDealt, int R>
__device__ __forceinline__ void read_frag(const lds8* tile, int first, int f, intx4 (&v)[2]) {
  const int i = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  constexpr int es = elem_size(kT), kPieces = kOuter ? R * es / 16 : 8;
  typedef __attribute__((address_space(3))) const intx4 piece;
  if constexpr (!kOuter) {
    // a fragment's rows all have the swizzle of the lane's first one
    const int r = first + frag_row<kDealt>(0, i), at = r * kStepBytes + ((g ^ swizzle<kT, kOuter, kDealt, kPieces>(r)) << 4);
    const int to = frag_row<kDealt>(f, 0) * kStepBytes;
    v[0] = *reinterpret_cast<piece*>(tile + at + to);
    v[1] = *reinterpret_cast<piece*>(tile + (at ^ 64) + to);
  } else if constexpr (kT == kF32) {
    const int col = first + frag_row<kDealt>(f, i);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = h * 16 + g * 4 + e;
        const int at = k * R * 4 + (((col >> 2) ^ swizzle<kT, kOuter, kDealt, kPieces>(k)) << 4) + (col & 3) * 4;
        v[h][e] = *reinterpret_cast<__attribute__((address_space(3))) const int*>(tile + at);
      }
  } else {
    // the transposing read: 16 lanes give the addresses of 4 values of k times 16 columns, lane j those of value j / 4
    // and columns 4 (j % 4) .. + 3, and lane i gets column i's four values
    const int col = first + frag_row<kDealt>(f, (i & 3) * 4);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      shortx4 t[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int k = h * 32 + g * 8 + e * 4 + (i >> 2);
        const int at = k * R * 2 + (((col >> 3) ^ swizzle<kT, kOuter, kDealt, kPieces>(k)) << 4) + (col & 7) * 2;
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
  // Pieces by integer arithmetic: the first is x cut to bf16 (rounded it would be infinite for the largest of fp32), the
  // second rounded (halves away from zero), the last exact.  10,000 rows over 6 experts, 1024 x 1024: 134 us, with the first
  // rounded too 139, with the conversion instruction 152; the error against 64 bits is the rounded one's within 1%.
  __device__ __forceinline__ void take(const intx4 (&u)[2]) {
    uint32_t w[3][4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      uint32_t x[3][2];
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        const uint32_t v = (uint32_t)(int)u[(e + d) >> 2][(e + d) & 3];
        x[0][d] = v & 0xffff0000u;
        const float r1 = __builtin_bit_cast(float, v) - __builtin_bit_cast(float, x[0][d]);
        x[1][d] = (__builtin_bit_cast(uint32_t, r1) + 0x8000u) & 0xffff0000u;
        x[2][d] = __builtin_bit_cast(uint32_t, r1 - __builtin_bit_cast(float, x[1][d]));
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) w[k][e >> 1] = __builtin_amdgcn_perm(x[k][1], x[k][0], 0x07060302u);   // the upper halves
    }
#pragma unroll
    for (int k = 0; k < 3; ++k)
      p[k] = __builtin_bit_cast(bf16x8, intx4{(int)w[k][0], (int)w[k][1], (int)w[k][2], (int)w[k][3]});
  }
};

// The matrix instructions of a product of fragments, one after another on the same accumulator: part q of kParts.
template <int kT>
constexpr int kParts = kT == kE4m3 ? 1 : kT == kF32 ? 6 : 2;
// sb, sa: four scale bytes each, of which kSB and kSA are the fragments'.
template <int kT, int kSB, int kSA, int q>
__device__ __forceinline__ floatx4 multiply(const Frag<kT>& b, const Frag<kT>& a, floatx4 c, int sb, int sa) {
  if constexpr (kT == kE4m3) {
    const intx8 x = __builtin_shufflevector(b.v[0], b.v[1], 0, 1, 2, 3, 4, 5, 6, 7);
    const intx8 y = __builtin_shufflevector(a.v[0], a.v[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 0, 0, kSB, sb, kSA, sa);
  } else if constexpr (kT == kF32) {
    constexpr int pb[6] = {2, 1, 0, 1, 0, 0}, pa[6] = {0, 1, 2, 0, 1, 0};      // the smallest first
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.p[pb[q]], a.p[pa[q]], c, 0, 0, 0);
  } else if constexpr (kT == kBf16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b.v[q]), __builtin_bit_cast(bf16x8, a.v[q]), c,
                                                   0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b.v[q]), __builtin_bit_cast(f16x8, a.v[q]), c,
                                                  0, 0, 0);
  }
}

// Expert e's rows.
__device__ __forceinline__ void expert_rows(Args& P, int total, int e, int& s, int& t) {
  s = min(max(P.offsets[e], 0), total);
  t = min(max(P.offsets[e + 1], s), total);
}

struct Tile {
  int e, row0, rows, n0;           // rows row0 .. row0 + rows belong to the tile's expert from the tile's first on
  int steps, length;               // of its part of the reduction
  int tail;                        // the step in which k ends inside a 16-byte piece, or -1
  bool any;
};

// The workgroup's tiles, one after another.  Every XCD takes a consecutive part of the list, so that tiles that share rows
// or columns share its L2; its workgroups take neighbouring tiles at a time.  kRed: tiles of different experts differ in
// length, so each XCD takes shares of many experts (16,384 rows unevenly over 32 experts of 1408 x 2048 bf16: 139 us, with
// consecutive experts 160; over 8 of 1536 x 2048 153 and 225; evenly over 32 127 and 124).
template <int kGroup, int BM, int BN>
struct Tiles {
  int at, end, stride;             // in the list
  int s, t, count, incl;           // kRows: lane l's expert, if there are at most 64: rows s .. t, tiles, tiles up to its last

  // The lane's expert of those from e0 on, with `before` tiles in front.
  __device__ __forceinline__ void part(Args& P, int e0, int before) {
    const int lane = threadIdx.x & 63;
    s = t = 0;
    if (e0 + lane < P.groups) expert_rows(P, P.m, e0 + lane, s, t);
    incl = count = (t - s + BM - 1) / BM;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(incl, o, 64);
      if (lane >= o) incl += v;
    }
    incl += before;
  }

  __device__ __forceinline__ void start(Args& P) {
    const int xcd = (int)blockIdx.x % kXcd;
    at = (int)blockIdx.x / kXcd;
    stride = (int)gridDim.x / kXcd;
    if constexpr (kGroup == kRed) {
      const int shares = (P.tiles_m * P.tiles_n + P.share - 1) / P.share * P.groups;
      end = uniform(shares > xcd ? (shares - xcd + kXcd - 1) / kXcd * P.share : 0);
      return;
    }
    int total = P.tiles_m;
    if constexpr (kGroup == kRows) {
      total = 0;
      for (int e0 = 0; e0 < P.groups; e0 += 64) {
        part(P, e0, total);
        total = uniform(__shfl(incl, 63, 64));
      }
    }
    total *= P.tiles_n;
    total = uniform(total);
    const int per = (total + kXcd - 1) / kXcd, first = xcd * per;
    at += first;
    end = min(first + per, total);
  }

  // Tile id of `high` rows of tiles: eight rows at a time, column by column, so that the 32 tiles that an XCD works on at
  // once read 8 tiles of one operand and 4 of the other.
  __device__ __forceinline__ static void place(Args& P, int id, int high, Tile& T) {
    const int block = 8 * P.tiles_n, b = uniform(id / block), in = id - b * block, rows = min(high - b * 8, 8);
    const int nt = uniform(in / rows);
    T.n0 = nt * BN;
    T.row0 = (b * 8 + in - nt * rows) * BM;
  }

  __device__ __forceinline__ Tile next(Args& P) {
    Tile T;
    T.e = T.row0 = T.rows = T.n0 = T.steps = T.length = 0;
    T.tail = -1;
    int id = at;
    if constexpr (kGroup == kRed) {
      // every eighth of the list of all experts' shares is the XCD's; the last one of an expert may be shorter
      const int all = P.tiles_m * P.tiles_n, share = P.share, shares = (all + share - 1) / share;
      for (id = all; at < end && id >= all; at += stride) {
        const int q = at / share, of = (int)blockIdx.x % kXcd + q * kXcd;
        T.e = uniform(of / shares);
        id = uniform((of - T.e * shares) * share + at - q * share);
      }
      T.any = id < all;
    } else {
      T.any = at < end;
      at += stride;
    }
    if (!T.any) return T;
    if constexpr (kGroup == kRows) {
      const int mt = uniform(id / P.tiles_n), all = P.groups;
      int before = 0;
      for (int e0 = 0; e0 < all; e0 += 64) {
        if (all > 64) part(P, e0, before);
        const uint64_t hit = __ballot(incl > mt);
        if (hit) {
          const int h = __builtin_ctzll(hit);
          const int high = uniform(__shfl(count, h, 64)), first = uniform(__shfl(incl, h, 64)) - high;
          T.e = uniform(e0 + h);
          // offsets that decrease give experts the same rows: the sum may pass 2^31, the tile stays one of its expert's
          place(P, min(max(id - first * P.tiles_n, 0), high * P.tiles_n - 1), high, T);
          T.row0 += uniform(__shfl(s, h, 64));
          T.rows = uniform(__shfl(t, h, 64)) - T.row0;
          break;
        }
        before = __shfl(incl, 63, 64);
      }
    } else {
      place(P, id, P.tiles_m, T);
      T.rows = P.m - T.row0;
    }
    return T;
  }
};

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
__device__ __forceinline__ void put(void* y, int64_t at, int c, int n, bool aligned, int type, const float (&v)[kN]) {
  if (type == E2V2_F32) put_row<float, kN>(static_cast<float*>(y) + at, c, n, aligned, v);
  else if (type == E2V2_BF16) put_row<__bf16, kN>(static_cast<__bf16*>(y) + at, c, n, aligned, v);
  else put_row<_Float16, kN>(static_cast<_Float16*>(y) + at, c, n, aligned, v);
}

// Zeros in the rows of y that belong to no expert, those before the first one's and behind the last one's.
__device__ __forceinline__ void fill_rows(Args& P) {
  int s, t, last;
  expert_rows(P, P.m, 0, s, t);
  expert_rows(P, P.m, P.groups - 1, t, last);
  const int size = P.out_type == E2V2_F32 ? 4 : 2, first = s, rows = s + P.m - max(last, s);
  uint8_t* y = static_cast<uint8_t*>(P.y);
  const bool wide = (((uint64_t)y | (uint64_t)(P.ldy * size) | (uint64_t)(P.n * size)) & 15) == 0;
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    uint8_t* row = y + (int64_t)(r < first ? r : P.m - rows + r) * P.ldy * size;
    if (wide) {
      for (int c = threadIdx.x; c < P.n * size / 16; c += blockDim.x) reinterpret_cast<uint4*>(row)[c] = make_uint4(0, 0, 0, 0);
    } else {
      for (int c = threadIdx.x; c < P.n * size / 2; c += blockDim.x) reinterpret_cast<uint16_t*>(row)[c] = 0;
    }
  }
}

// kAO, kBO: outer layout of a, b.  WM x WN wavefronts.  A workgroup takes one tile after another, and the steps of all its
// tiles are one pipeline.  A wavefront holds a step's b and half of its a in registers.  In a step's first half it reads
// the other half of a and multiplies with the first; in the second half it multiplies with the other, and reads the first
// half of a and, behind the last products that need it, each fragment of b of the next step.  The loads of the step after
// the next go into this step's tiles as soon as all have read them (b and the first half of a in the first half of the
// step, the rest in the second), between the products, and are waited for more than a step later.  Products stand on both
// sides of the two barriers of a step.
//
// Bound: the matrix units' issue and the loads into LDS.  8192 x 8192 x 4096: e4m3 239 us (2.30 PFLOP/s, matrix units 49%
// busy), bf16 417 forward, 411 rows' gradient, 424 weights' (1.30 to 1.34 PFLOP/s, 55 to 58%).  8192^3 bf16: a step's loads in
// one clump behind one barrier 977 us, sent between the products with descriptors kept 856, and sent into each half of a tile
// as soon as it is free 794.  A change of tiles costs 8 us, 6.7 of which its stores take at 5 TB/s.
template <int kT, bool kAO, bool kBO, int BM, int BN, int WM, int WN, int kGroup, bool kStaged>
__global__ __launch_bounds__(WM * WN * 64, 2) void k_mm(MmArgs) {
  constexpr int NT = WM * WN * 64, FM = BM / WM / 16, FN = BN / WN / 16, FH = FM / 2;
  constexpr int es = elem_size(kT), kK = kStepBytes / es, kTile = (BM + BN) * kStepBytes;
  constexpr bool k8 = kT == kE4m3;
  __shared__ __attribute__((aligned(1024))) uint8_t mem[2 * kTile + (k8 ? 4 * NT * 4 : 0)];
  if constexpr (kGroup == kRows) {
    if (arguments().fill) fill_rows(arguments());
  }
  const int wave = uniform((int)threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  const int i = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  typedef TileLoad<kT, kAO, false, BM, NT, kStaged> LoadA;
  typedef TileLoad<kT, kBO, true, BN, NT, kStaged> LoadB;
  LoadA la;
  LoadB lb;
  ScaleLoad<BM, BN, NT> ls;
  Tiles<kGroup, BM, BN> tiles;
  tiles.start(arguments());

  // The next tile of the list, its loads prepared.  Every tile has as many steps as are on their way at once, so that they
  // are those of two tiles at most; what goes past its reduction is zeros.
  constexpr int kAhead = kStaged ? 3 : 2;
  auto next_tile = [&]() -> Tile {
    Args& P = arguments();
    Tile T = tiles.next(P);
    if (!T.any) return T;
    int k0 = 0, k1 = P.k;
    if constexpr (kGroup == kRed) expert_rows(P, P.k, T.e, k0, k1);
    if (P.splits > 1) {
      const int steps = (k1 - k0 + kK - 1) / kK, each = uniform((steps + P.splits - 1) / P.splits) * kK;
      k1 = min(k1, k0 + ((int)blockIdx.y + 1) * each);
      k0 = min(k0 + (int)blockIdx.y * each, k1);
    }
    k0 = uniform(k0);
    T.length = uniform(k1) - k0;
    T.steps = max((T.length + kK - 1) / kK, kAhead);
    if (!kStaged && !(kAO && kBO) && ((T.length * es) & 15)) T.tail = T.length / kK;
    const uint8_t* pb = P.b + (kGroup == kRows ? (int64_t)T.e * P.b_group : 0);
    if constexpr (kAO) la.start(P.a + (int64_t)k0 * P.lda + (int64_t)T.row0 * es, (int)P.lda, T.rows, T.length);
    else la.start(P.a + (int64_t)T.row0 * P.lda + (int64_t)k0 * es, (int)P.lda, T.rows, T.length);
    if constexpr (kBO) lb.start(pb + (int64_t)k0 * P.ldb + (int64_t)T.n0 * es, (int)P.ldb, P.n - T.n0, T.length);
    else lb.start(pb + (int64_t)T.n0 * P.ldb + (int64_t)k0 * es, (int)P.ldb, P.n - T.n0, T.length);
    if constexpr (k8) {
      const int b0 = k0 / 128, blocks = (T.length + 127) / 128;
      if (wave * 64 < BM) {
        ls.start(P.sa + (int64_t)T.row0 * P.sa_ld + b0 * P.sa_k, P.sa_ld, P.sa_k, min(T.rows, BM), blocks, 1);
      } else {
        const uint8_t* ps = P.sb + (kGroup == kRows ? (int64_t)T.e * P.sb_group : 0);
        // a tile of 64 lies inside one block of the 128 rows that share a scale, larger ones hold whole blocks
        ls.start(ps + (int64_t)(P.sb_rows > 1 ? T.n0 / 128 : T.n0) * P.sb_ld + b0 * P.sb_k, P.sb_ld, P.sb_k,
                 min(P.n - T.n0, BN), blocks, P.sb_rows > 1 ? 128 : 1);
      }
    }
    return T;
  };

  auto buf = [&](int c) { return (lds8*)mem + (c & 1) * kTile; };
  lds8* const ring = (lds8*)mem + 2 * kTile;

  // The tile that is computed, the one behind it, and the step that is sent next.
  Tile now = next_tile(), then = now;
  if (!now.any) return;
  then.any = false;
  int ft = 0, fc = 0, fsteps = now.steps;
  const int mem0 = uniform((int)(uintptr_t)(lds8*)mem + wave * 1024), ring0 = uniform((int)(uintptr_t)ring + wave * 256);
  constexpr int kRa = LoadA::kRounds, kRb = LoadB::kRounds;
  auto prepare = [&] {
    if (ft == fsteps) {
      then = next_tile();
      ft = 0;
      fsteps = then.any ? then.steps : INT32_MAX;
      if (!then.any) la.stop(), lb.stop(), ls.stop();
    }
    la.prepare(ft);
    lb.prepare(ft);
  };
  // Even rounds of an inner a are the first half of each wavefront's rows, odd ones the other half; all rounds of an outer a
  // are needed by both.  Piece p of what the first and the second half of a step send:
  constexpr bool kHalves = !kAO;
  static_assert(!kHalves || BM / WM / 2 == NT / 8, "a round is half of a wavefront's rows");
  constexpr int kSend1 = kStaged ? 0 : k8 + kRb + (kHalves ? kRa / 2 : 0), kSend2 = kStaged ? 1 : kHalves ? kRa / 2 : kRa;
  auto send1 = [&](auto p) {
    const int to = mem0 + (fc & 1) * kTile;
    if constexpr (p < k8) ls.send(ft, fc, ring0);
    else if constexpr (p < k8 + kRb) lb.template send<p - k8>(to + BM * kStepBytes);
    else if constexpr (p < kSend1) la.template send<2 * (p - k8 - kRb)>(to);
  };
  auto send2 = [&](auto p) {
    if constexpr (kStaged && p == 0) {
      if constexpr (k8) ls.send(ft, fc, ring0);
      la.take(ft);
      lb.take(ft);
    } else if constexpr (p < kSend2) {
      la.template send<kHalves ? 2 * p + 1 : p>(mem0 + (fc & 1) * kTile);
    }
  };
  auto send = [&] {
    prepare();
    each<kSend1>(send1);
    each<kSend2>(send2);
    ++ft, ++fc;
  };
  // Waits until all but the last kLeft loads and stores are done and all LDS reads, and meets the others.
  auto meet = [](auto left) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((int)left) : "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr std::integral_constant<int, 0> kNone{};
  // From registers into the tiles of step c: what was sent last.
  auto put_held = [&](int c) {
    if constexpr (kStaged) {
      la.put(buf(c));
      lb.put(buf(c) + BM * kStepBytes);
    }
  };
  // Step t of a tile, step c of all: clears what lies behind the end of k.
  auto clear = [&](int t, int tail, int length, int c) {
    if constexpr (!kStaged && !(kAO && kBO)) {
      if (t == tail) {
        meet(kNone);                               // what is cleared has arrived, for all
        LoadA::clear_tail(length * es - t * kStepBytes, buf(c));
        LoadB::clear_tail(length * es - t * kStepBytes, buf(c) + BM * kStepBytes);
        meet(kNone);
      }
    }
  };

  Frag<kT> fa[2][FH], fb[FN];
  int sa[2], sb;                                   // scale bytes of the fragments, four in a dword
  static_assert(FH <= 4 && FN == 4, "a byte a fragment");
  auto scale = [&](int c, int row) {
    return *reinterpret_cast<__attribute__((address_space(3))) const int*>(ring + (c & 3) * NT * 4 + row * 4);
  };
  auto read_a = [&](int c, int half) {
    int u8 = 0;
#pragma unroll
    for (int f = 0; f < FH; ++f) {
      intx4 u[2];
      read_frag<kT, kAO, false, BM>(buf(c), wm * FM * 16, half * FH + f, u);
      fa[half][f].take(u);
      if constexpr (k8) u8 |= scale(c, wm * FM * 16 + (half * FH + f) * 16 + i) << (8 * f);
    }
    sa[half] = u8;
  };
  auto read_b = [&](int c, int h) {
    intx4 u[2];
    read_frag<kT, kBO, true, BN>(buf(c) + BM * kStepBytes, wn * FN * 16, h, u);
    fb[h].take(u);
  };
  auto read_sb = [&](int c) {
    int u8 = 0;
    if constexpr (k8) {
#pragma unroll
      for (int h = 0; h < FN; ++h) u8 |= scale(c, BM + wn * FN * 16 + frag_row<true>(h, i)) << (8 * h);
    }
    return u8;
  };

  send();
  put_held(0);
  send();
  if constexpr (kStaged) {
    put_held(1);
    send();
    meet(kNone);
  } else {
    meet(std::integral_constant<int, kSend1 + kSend2>{});
  }
  clear(0, now.tail, now.length, 0);
  read_a(0, 0);
#pragma unroll
  for (int h = 0; h < FN; ++h) read_b(0, h);
  sb = read_sb(0);

  // loads that may be on their way at the barriers: those of half a step and of a whole one; behind a whole tile FM FN / 2
  // stores of 16 bytes at least besides, which need not have ended in the first step and at the next one's beginning (in
  // the kernels of 256 with experts most have: they reload spilled registers between the stores, which waits for all before)
  constexpr int kWhole = kStaged ? 0 : kSend1 + kSend2, kMid = kStaged ? 0 : kHalves ? kWhole : kSend1;
  constexpr int kStores = kStaged ? 0 : FM * FN / 2;
  constexpr int kPer1 = (kSend1 + 1) / 2, kPer2 = (kSend2 + 1) / 2;      // loads behind each two of b's fragments
  int c = 0;                                       // steps done, of all tiles
  bool stored = false;
  while (true) {
    floatx4 acc[FM][FN];
#pragma unroll
    for (int f = 0; f < FM; ++f)
#pragma unroll
      for (int h = 0; h < FN; ++h) acc[f][h] = floatx4{0.f, 0.f, 0.f, 0.f};
    // A half of a with two fragments of b: the chains of each accumulator's instructions side by side.
    auto products = [&](auto half, auto n) {
      each<kParts<kT>>([&](auto q) {
        each<2>([&](auto h) {
          each<FH>([&](auto f) {
            constexpr int b = 2 * n + h, at = half * FH + f;
            acc[at][b] = multiply<kT, b, f, q>(fb[b], fa[half][f], acc[at][b], sb, sa[half]);
          });
        });
      });
    };
    for (int t = 0; t < now.steps; ++t, ++c) {
      prepare();
      if (stored && t < 2) meet(std::integral_constant<int, kWhole + kStores>{});
      else meet(std::integral_constant<int, kWhole>{});
      read_a(c, 1);
      each<2>([&](auto n) {
        products(std::integral_constant<int, 0>{}, n);
        __builtin_amdgcn_sched_barrier(0);
        each<kPer1>([&](auto p) { send1(std::integral_constant<int, n * kPer1 + p>{}); });
      });
      // the products stay in front of the barrier: the compiler moved them behind the branch there
#pragma unroll
      for (int f = 0; f < FH; ++f)
#pragma unroll
        for (int h = 0; h < FN; ++h) asm volatile("" : "+v"(acc[f][h]));
      if (stored && t == 0) meet(std::integral_constant<int, kMid + kStores>{});
      else meet(std::integral_constant<int, kMid>{});
      put_held(c);
      const bool in = t + 1 < now.steps;
      clear(in ? t + 1 : 0, in ? now.tail : then.tail, in ? now.length : then.length, c + 1);
      read_a(c + 1, 0);                            // behind the last step: what lies there is not used
      const int next_sb = read_sb(c + 1);
      each<2>([&](auto n) {
        products(std::integral_constant<int, 1>{}, n);
        __builtin_amdgcn_sched_barrier(0);         // the fragments' registers are free here, and taken at once
        read_b(c + 1, 2 * n);
        read_b(c + 1, 2 * n + 1);
        each<kPer2>([&](auto p) { send2(std::integral_constant<int, n * kPer2 + p>{}); });
      });
      sb = next_sb;
      ++ft, ++fc;
    }

    // lane (g, i) holds row i of each fragment and eight columns of it for each two of b's
    Args& P = arguments();
    const int col = now.n0 + wn * FN * 16 + g * 8;
    const int64_t plane = kGroup == kRed ? now.e : 0;
    const bool part = P.splits > 1;
    void* y = part ? P.part : P.y;
    const int64_t ld = part ? P.n : P.ldy;
    const int type = part ? E2V2_F32 : P.out_type;
    const int64_t row0 = (part ? (int64_t)blockIdx.y * (kGroup == kRed ? P.groups : 1) + plane : plane) * P.m + now.row0;
    const bool aligned = (((uint64_t)y | (uint64_t)(ld * (type == E2V2_F32 ? 4 : 2))) & 15) == 0;
#pragma unroll
    for (int f = 0; f < FM; ++f) {
      const int r = wm * FM * 16 + f * 16 + i;
      if (r >= now.rows) continue;
#pragma unroll
      for (int h = 0; h < FN; h += 2) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[f][h + e / 4][e % 4];
        put<8>(y, (row0 + r) * ld, col + h * 16, P.n, aligned, type, v);
      }
    }
    if (!then.any) return;
    stored = aligned && now.rows >= BM && now.n0 + BN <= P.n;      // then FM FN / 2 stores of 16 bytes at least
    now = then;
    then.any = false;
    then.tail = -1;
  }
}

// Few rows (16 of one expert in a workgroup): a pass over b's bytes.  A workgroup takes 16 columns of y, each of its 8
// wavefronts an eighth of k, read from memory straight into the registers that the matrix instructions take, four steps
// at a time (32 KB a workgroup on the way); the eighths are added in order through LDS.  Inner operands whose rows start on
// 16 bytes.  Bound: HBM for many experts, latency for one matrix: 13 rows of 64 experts of 1024 x 2048 bf16 (46 MB) 14.6 us,
// 3.2 TB/s; 4096 x 4096 e4m3, one row, 5 to 6 us.  Two or four fragments of rows at once were slower (their loads leave
// fewer steps in the registers): 32 rows are two workgroups, the second of which finds b in L2.
constexpr int kThinWaves = 8, kThinSide = 16;

template <int kT, int kGroup>
__global__ __launch_bounds__(64 * kThinWaves, 4) void k_thin(MmArgs) {
  constexpr int es = elem_size(kT), kUnroll = 4;
  constexpr bool k8 = kT == kE4m3;
  __shared__ floatx4 sums[kThinWaves][64];
  if constexpr (kGroup == kRows) {
    if (arguments().fill) fill_rows(arguments());
  }
  Args& P = arguments();
  Tiles<kGroup, kThinSide, kThinSide> tiles;
  tiles.start(P);
  const int wave = uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int width = P.k * es, all = (width + kStepBytes - 1) / kStepBytes, each_ = (all + kThinWaves - 1) / kThinWaves;
  const int t0 = wave * each_, t1 = min(t0 + each_, all);
  for (Tile T = tiles.next(P); T.any; T = tiles.next(P)) {
    const int rows = min(T.rows, kThinSide), cols = min(P.n - T.n0, kThinSide), r = min(i, rows - 1), c = min(i, cols - 1);
    auto buffer = [&](const uint8_t* p, int64_t ld, int n) {
      return __builtin_amdgcn_make_buffer_rsrc((void*)uniform(p), 0, uniform(((n - 1) * (int)ld + width + 15) & ~15),
                                               0x00020000);
    };
    const auto ra = buffer(P.a + (int64_t)T.row0 * P.lda, P.lda, rows);
    const auto rb = buffer(P.b + (kGroup == kRows ? (int64_t)T.e * P.b_group : 0) + (int64_t)T.n0 * P.ldb, P.ldb, cols);
    const unsigned oa = (unsigned)(r * (int)P.lda + g * 16), ob = (unsigned)(c * (int)P.ldb + g * 16);
    const uint8_t *pa = P.sa, *pb = P.sb;
    if constexpr (k8) {
      const int col = T.n0 + c;
      pa += (int64_t)(T.row0 + r) * P.sa_ld;
      pb += (kGroup == kRows ? (int64_t)T.e * P.sb_group : 0) + (int64_t)(P.sb_rows > 1 ? col / 128 : col) * P.sb_ld;
    }
    floatx4 acc = floatx4{0.f, 0.f, 0.f, 0.f};
    for (int t = t0; t < t1; t += kUnroll) {
      intx4 ub[kUnroll][2], ua[kUnroll][2];
      int sb[kUnroll], sa[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int at = (t + u) * kStepBytes + g * 16;        // the lane's first piece; the other lies 64 bytes further
        const bool in = t + u < t1, in0 = in && at < width, in1 = in && at + 64 < width;
        const unsigned k = (unsigned)((t + u) * kStepBytes);
        ub[u][0] = __builtin_amdgcn_raw_buffer_load_b128(rb, in0 ? ob + k : kNowhere, 0, 0);
        ub[u][1] = __builtin_amdgcn_raw_buffer_load_b128(rb, in1 ? ob + k + 64 : kNowhere, 0, 0);
        ua[u][0] = __builtin_amdgcn_raw_buffer_load_b128(ra, in0 ? oa + k : kNowhere, 0, 0);
        ua[u][1] = __builtin_amdgcn_raw_buffer_load_b128(ra, in1 ? oa + k + 64 : kNowhere, 0, 0);
        sb[u] = sa[u] = 0;
        if constexpr (k8) {
          const int64_t block = min(t + u, t1 - 1);
          sb[u] = pb[block * P.sb_k];
          sa[u] = pa[block * P.sa_k];
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        auto clear = [&](intx4 (&v)[2]) {                    // the bytes behind the end of k
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            const int h = width - ((t + u) * kStepBytes + g * 16 + (d >> 2) * 64 + (d & 3) * 4);
            v[d >> 2][d & 3] = h >= 4 ? v[d >> 2][d & 3] : h <= 0 ? 0 : v[d >> 2][d & 3] & (int)((1u << (8 * h)) - 1u);
          }
        };
        if ((width & 15) && (t + u + 1) * kStepBytes > width) clear(ub[u]), clear(ua[u]);
        Frag<kT> fa, fb;
        fb.take(ub[u]);
        fa.take(ua[u]);
        each<kParts<kT>>([&](auto q) { acc = multiply<kT, 0, 0, q>(fb, fa, acc, sb[u], sa[u]); });
      }
    }
    sums[wave][lane] = acc;
    __syncthreads();
    // lane (g, i) holds row i, columns 4 g .. 4 g + 3
    if (wave == 0 && i < rows) {
      floatx4 v = sums[0][lane];
#pragma unroll
      for (int w = 1; w < kThinWaves; ++w) v += sums[w][lane];
      const float o[4] = {v[0], v[1], v[2], v[3]};
      const int size = P.out_type == E2V2_F32 ? 4 : 2;
      const bool aligned = (((uint64_t)P.y | (uint64_t)(P.ldy * size)) & (4 * size - 1)) == 0;
      put<4>(P.y, (int64_t)(T.row0 + i) * P.ldy, T.n0 + g * 4, P.n, aligned, P.out_type, o);
    }
    __syncthreads();
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
  if constexpr (kGroup == kRows) tiles = (int64_t)(P.m / BM + (P.groups < P.m ? P.groups : P.m)) * P.tiles_n;
  else tiles = (int64_t)P.tiles_m * P.tiles_n;
  if constexpr (kGroup == kRed) {
    // Shares of 32 tiles, which read 8 tiles of one operand and 4 of the other, but four of them for each XCD, as experts
    // differ in length; and a workgroup for each tile of the XCD that has most.
    const int64_t cut = std::min<int64_t>(kXcd, std::max<int64_t>({1, 4 * kXcd / P.groups, tiles / 32}));
    P.share = (int)((tiles + cut - 1) / cut);
    const int64_t shares = (tiles + P.share - 1) / P.share * P.groups;
    tiles = (shares + kXcd - 1) / kXcd * P.share * kXcd;
  }
  tiles = (tiles + kXcd - 1) / kXcd * kXcd;
  constexpr int64_t kSlots = 256 * (BM == 256 ? 1 : BM == 128 ? 2 : 4);     // workgroups that the 256 CUs hold
  tiles = tiles < kSlots ? tiles : kSlots;
  hipLaunchKernelGGL((k_mm<kT, kAO, kBO, BM, BN, WM, WN, kGroup, kStaged>), dim3((unsigned)tiles, (unsigned)P.splits),
                     dim3(WM * WN * 64), 0, s, P);
}

// Whether few rows meet so few bytes of b that the pass over them is the shorter way: each 16 rows of an expert read its
// matrix once more (from L2), and every 16 columns all of the rows.  A limit where both take as long: one row of 64 experts
// of 1024 x 2048 bf16 (268 MB) 42 us and 33 with tiles, 13 rows 14 and 23; e4m3 8192 x 8192 (67 MB), 4 rows 15 and 18, 16
// rows 21 and 18; 4096 x 4096, 1 row 5 and 11, 32 rows 15 and 12.
inline bool thin_rows(int64_t m, int64_t n, int64_t k_bytes, int groups) {
  const int64_t each = (m + groups - 1) / groups, tiles = (each + 15) / 16;
  if (each > 64) return false;
  const int64_t read = (groups < m ? groups : m) * n * k_bytes * tiles * (16 + (each < 16 ? each : 16)) / 16;
  return read <= (tiles == 1 ? 100 : 40) * 1000000LL;
}

template <int kT, int kGroup>
void launch_thin(MmArgs P, hipStream_t s) {
  P.tiles_n = (P.n + kThinSide - 1) / kThinSide;
  P.tiles_m = (P.m + kThinSide - 1) / kThinSide;
  P.splits = 1;
  int64_t tiles = (kGroup == kRows ? P.m / kThinSide + (P.groups < P.m ? P.groups : P.m) : P.tiles_m) * (int64_t)P.tiles_n;
  tiles = (tiles + kXcd - 1) / kXcd * kXcd;
  tiles = tiles < 8192 ? tiles : 8192;
  hipLaunchKernelGGL((k_thin<kT, kGroup>), dim3((unsigned)tiles), dim3(64 * kThinWaves), 0, s, P);
}

inline void launch_mm_sum(const MmArgs& P, int64_t rows, hipStream_t s) {
  const int64_t blocks = (rows * P.n + 255) / 256;
  hipLaunchKernelGGL(k_mm_sum, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, P.part, P.splits, rows,
                     P.n, P.y, P.ldy, P.out_type);
}

}  // namespace
}  // namespace e2v2
