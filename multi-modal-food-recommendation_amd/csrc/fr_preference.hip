// Log-probabilities of items under a softmax over the whole item table, with gradients, and the
// preference loss (paired log ratios) over lists of them.  The score matrix is never stored.
//
//   z[n, v] = c <H[n], W[v]>,  lse[n] = log sum_v exp z[n, v],  logp[n] = z[n, t_n] - lse[n]
//   p = exp(z - lse);  dH[n] = a_n c ((1 - p[n, t_n]) W[t_n] - o[n]),  o[n] = sum_{v != t_n} p[n, v] W[v]
//   dW = g^T H,  g[n, v] = a_n c ([v = t_n] - p[n, v])         (a = the upstream gradient of logp)
//
// o does not depend on a: where dH will be asked for, the forward adds it up along with the statistics, from
// the same scores, and the backward of H is left with a row operation.  The target is kept apart in both,
// so that 1 - p and logp of a nearly certain item keep their precision.
//
// All three products run on the matrix cores in tiles of 32 x 32 scores, one side's rows (X) as B
// operands in registers, the other's (Y) as A operands from LDS:
//
//   S = Y X^T          lane l holds X row l % 32 and Y rows i(r, h) = 8 (r / 4) + 4 h + r % 4 for its 16
//                      results r and half h = l / 32: softmax statistics stay inside a lane
//   out^T += Y^T G     the results, turned into g, ARE the B operand of the second product (its k slots
//                      are Y rows in the order i(r, h)), so g never leaves the registers; the A operand
//                      is the same Y tile read by columns (transposing LDS reads in bf16)
//
// The forward has X = users, Y = items, G = exp(z - running maximum) and out = o; dW has X = items, Y = users.
// The scores are computed once more for it (2 n v d flops of recomputation instead of n v stored scores).
// o's running maximum is raised only when a score exceeds it by 2^8 (exp then stays below 256), since that
// rescales the accumulators.
// Long axes are split over workgroups; partials are joined in a fixed order, no float atomics.
//
// bf16 tables are multiplied as they are (products exact, sums fp32).  fp32 tables are multiplied in parts:
//
//   scores   x = 2^-e (x0 + x1), two fp16 parts of 11 bits each, e shared by 32 rows so that their largest
//            entry is in [2^13, 2^14): the products 00, 01, 10 leave 2^-22 of |x||y| (an fp32 sum of 64
//            products leaves as much), and 2^-38 of the 32 rows' largest entry for those far below it, which
//            is kept below 2^-23 of a score by kPartsLimit
//   g W, g H x = x0 + x1 + x2, three bf16 parts of 8 bits, which keep fp32's range (g spans many orders):
//            the six products of parts down to 2^-18 of the largest; the dropped ones are below 2^-26
//
// which is 9 instructions of 32 x 32 x 16 per 16 columns of both products, instead of 16 fp32 ones of twice
// the length.  From d = 65 on the five parts of a tile leave LDS for one workgroup per unit (or none), and the
// scores that go with a second product are computed from its three bf16 parts, too.  Blocks whose rows differ too
// much for the fp16 parts, with an infinite entry or one above 2^58 for the bf16 ones, get their scores from the fp32
// rows on the fp32 instruction (7,168 x 45,630 x 64: pass 0.73 ms without such items, 1.1 with one in 1,000 masked by
// -1e9, 1.3 with one in 100 = 28 % of the blocks, 1.9 where every block is one).  For bf16 tables G is rounded to bf16 (2^-9 of each term, about the
// rounding of the result itself), but for the target's entry, which outweighs the others in dW: it is taken in two
// parts (so is 1 - p, in fp32, in dH).  a_n and c are applied to g in dW and to the sum, in fp32, in dH.
//
// LDS: a row is CH chunks of 16 bytes, chunk c of row y at c ^ swz(y), so that both the row reads (32
// rows, one chunk column) and the column reads (8 rows, 4 neighbouring chunks) meet every bank
// equally (no bank conflicts counted).  Tiles go from memory to LDS without registers, two in turn, one
// barrier per tile.
//
// Bound by the matrix cores at the clock that their power allows (1.7-1.9 GHz under load; a library product of
// 8192^3 in bf16 reaches 1,206 TFLOP/s).  Medians of 20 launches each under a kernel trace: 3,840 x 1M x 256 bf16
// statistics and o 3.24 ms (1,210 TFLOP/s), dW 3.31 ms (1,190), boxes differ by 5 %; 7,168 x 45,630 x 64 fp32 343 and
// 363 us (statistics, dH and dW took 0.45, 0.90 and 0.87 ms with fp32 instructions).  Statistics alone are bound by the
// vector work per score (exponential, multiply-add, sum, maximum: some 44 cycles per 64 scores, 32 of d = 128's
// products): 1,800 x 29,943 x 128 bf16 28 us, some 8 of them the start and the operands' loading; a call of 7,168 x
// 45,630 x 64 bf16 75 us.  The matrix cores are busy 53-60 % of the cycles; what helped beside the products was fewer
// instructions and registers around them (addresses as constants, -lse as the accumulators' start); reading further
// ahead, more tiles in flight, one block's scores computed beside the statistics of another, no scheduling fences and
// wave priorities changed nothing beyond 2 % or cost time.
// What is spilled with d = 256 (and d = 128 in fp32) is reloaded per tile or before the loops: 11 registers per tile of
// 32 rows in bf16 with o, 5 in dW; fp32 10 with o, and 2 in dW of d = 128.
#include "fr_vec.h"

#include <algorithm>

namespace {

using fr::bf16_t;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

#define FR_LDS __attribute__((address_space(3)))
#define FR_GLOBAL __attribute__((address_space(1)))

constexpr int kMaxD = 256;
constexpr float kLog2e = 1.4426950408889634f;

// Y rows per LDS tile: 16 to 24 KiB of `parts` parts, or 32 rows
constexpr int tile_rows(int D, int parts) {
  const int rows = (parts == 1 ? 8192 : parts == 2 ? 4096 : 2048) / D;
  return rows < 32 ? 32 : rows;
}

// the operands' parts, for the statistics (GRAD false) and for the gradients
template <typename T, int D, bool GRAD>
struct Geo {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr bool HALF = F32 && (!GRAD || D <= 64);      // scores from two fp16 parts
  static constexpr int NS = HALF ? 2 : F32 ? 3 : 1;            // parts of the score product, from part 0
  static constexpr int NG = F32 ? 3 : 1;                       // parts of the second product, from part G0
  static constexpr int G0 = HALF ? 2 : 0;
  static constexpr int P = HALF ? (GRAD ? 5 : 2) : NS;         // parts in memory and LDS
  static constexpr int CH = D / 8;                             // chunks per row of one part
  static constexpr int TY = tile_rows(D, P);
  static constexpr int SUBS = TY / 32;
  static constexpr int PART = TY * CH;                         // chunks of one part of a tile
  static constexpr int CHUNKS = P * PART;
};

// the products of N parts that are kept, the smallest first: part of A, part of B
template <int N>
struct Products;
template <>
struct Products<1> {
  static constexpr int N = 1;
  static constexpr int at[1][2] = {{0, 0}};
};
template <>
struct Products<2> {
  static constexpr int N = 3;
  static constexpr int at[3][2] = {{1, 0}, {0, 1}, {0, 0}};
};
template <>
struct Products<3> {
  static constexpr int N = 6;
  static constexpr int at[6][2] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};
};

template <int CH>
__device__ __forceinline__ int swz(int row) {
  if constexpr (CH >= 16) return (row & 3) << 2 | ((row >> 2) & 3);
  else if constexpr (CH == 8) return ((row >> 1) & 1) << 2 | ((row >> 2) & 3);
  else return (row >> 2) & 3;
}

__device__ __forceinline__ int result_row(int r, int half) { return 8 * (r / 4) + 4 * half + r % 4; }

__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// eight values as P vectors of bf16 parts
template <int P>
__device__ __forceinline__ void parts_of(const float (&v)[8], u32x4 (&out)[P]) {
  float r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = v[j];
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t u = fr::pack_bf16(r[2 * j], r[2 * j + 1]);
      out[p][j] = u;
      if (p + 1 < P) {
        r[2 * j] -= __uint_as_float(u << 16);
        r[2 * j + 1] -= __uint_as_float(u & 0xffff0000u);
      }
    }
}

// the same of a row's entries as they come: one that would round to infinity is cut to the largest bf16 number, an
// infinite one is in the first part alone
template <int P>
__device__ __forceinline__ void row_parts_of(const float (&v)[8], u32x4 (&out)[P]) {
  if constexpr (P == 1) {
    parts_of<1>(v, out);
  } else {
    float first[8], rest[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t u = __float_as_uint(v[j]), size = u & 0x7fffffffu;
      first[j] = size >= 0x7f7f8000u && size <= 0x7f800000u ? __uint_as_float(u & 0xffff0000u) : v[j];
      rest[j] = size == 0x7f800000u ? 0.f : v[j] - fr::to_f32(fr::from_f32<bf16_t>(first[j]));
    }
    u32x4 a[1], b[P - 1];
    parts_of<1>(first, a);
    parts_of<P - 1>(rest, b);
    out[0] = a[0];
#pragma unroll
    for (int p = 1; p < P; ++p) out[p] = b[p - 1];
  }
}

// eight values times `scale` as two vectors of fp16 parts
__device__ __forceinline__ void halves_of(const float (&v)[8], float scale, u32x4 (&out)[2]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const fr::f32x2 x = {v[2 * j] * scale, v[2 * j + 1] * scale};
    const f16x2 hi = __builtin_convertvector(x, f16x2);
    const f16x2 lo = __builtin_convertvector(x - __builtin_convertvector(hi, fr::f32x2), f16x2);
    out[0][j] = __builtin_bit_cast(uint32_t, hi);
    out[1][j] = __builtin_bit_cast(uint32_t, lo);
  }
}

// A tile's LDS address; the tiles are aligned to their rows' 16 CH bytes (512 at most), so that the chunk number
// can be put into an address by exclusive or.
__device__ __forceinline__ uint32_t lds_of(const u32x4* tile) { return (uint32_t)(uintptr_t)(const FR_LDS u32x4*)tile; }
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at) {
  return *(const FR_LDS V*)(uintptr_t)at;
}

// Tiles of TY rows of Y (P parts, `part` elements apart) into LDS; rows past the end repeat the last one (masked
// by the reader).  A workgroup's load q is the 256 chunks from 256 q on.  The swizzle repeats after 16 rows, so a
// thread's offsets repeat, too, but for whole rows, and a tile costs little more than its loads.
template <typename G>
struct Stage {
  static constexpr int Q = G::CHUNKS / 256, ROWS = 256 / G::CH, NOFF = ROWS < 16 ? 16 / ROWS : 1;
  static_assert(G::PART % 256 == 0, "a load lies in one part");
  const char* base;
  int64_t part_bytes, ny;
  int ld;
  uint32_t off[NOFF];

  static __device__ __forceinline__ int row_of(int q) { return (q * 256 % G::PART + (int)threadIdx.x) / G::CH; }
  __device__ __forceinline__ uint32_t offset(int q, int row) const {
    const int c = (int)(threadIdx.x % G::CH) ^ swz<G::CH>(row_of(q));
    return (uint32_t)(row * ld + c * 8) * 2;
  }
  __device__ __forceinline__ Stage(const bf16_t* Y, int64_t ld_, int64_t part, int64_t ny_)
      : base(reinterpret_cast<const char*>(Y)), part_bytes(part * 2), ny(ny_), ld((int)ld_) {
#pragma unroll
    for (int q = 0; q < NOFF; ++q) off[q] = offset(q, row_of(q));
  }
  __device__ __forceinline__ void load(int64_t t, u32x4* tile) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const char* p = base + t * G::TY * ld * 2;
    const bool whole = (t + 1) * G::TY <= ny;
    const int last = (int)min(ny - 1 - t * G::TY, (int64_t)G::TY);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const char* from = p + q * 256 / G::PART * part_bytes;
      uint32_t o;
      if (whole) {
        from += (int64_t)((q * 256 % G::PART / 256 - q % NOFF) * ROWS) * ld * 2;
        o = off[q % NOFF];
      } else {
        o = offset(q, min(row_of(q), last));
      }
      __builtin_amdgcn_global_load_lds((const FR_GLOBAL void*)(from + o), (FR_LDS void*)(tile + q * 256 + wave * 64), 16, 0,
                                       0);
    }
  }
};

// one 32-row block of X as B operands: chunk 2 kk + half of row x0 + lane % 32, from the parts' copies (rows past the
// end: the last one again, whose results are not written)
template <typename G>
__device__ __forceinline__ void load_x(const bf16_t* X, int64_t ld, int64_t part, int64_t nx, int64_t x0,
                                       u32x4 (&f)[G::NS][G::CH / 2]) {
  const int lane = threadIdx.x & 63;
  const bf16_t* row = X + min(x0 + (lane & 31), nx - 1) * ld + lane / 32 * 8;
#pragma unroll
  for (int p = 0; p < G::NS; ++p)
#pragma unroll
    for (int kk = 0; kk < G::CH / 2; ++kk) f[p][kk] = *reinterpret_cast<const u32x4*>(row + p * part + kk * 16);
}

// an infinity or NaN among the wave's operands of bf16 parts
template <int NS, int KK>
__device__ __forceinline__ bool has_no_number(const u32x4 (&f)[NS][KK]) {
  bool any = false;
#pragma unroll
  for (int p = 0; p < NS; ++p)
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        any |= (f[p][kk][j] & 0x7f80u) == 0x7f80u || (f[p][kk][j] & 0x7f800000u) == 0x7f800000u;
  return __ballot(any);
}

template <bool HALF>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 acc) {
  if constexpr (HALF)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0,
                                                   0, 0);
}

// N steps of products whose A operands come from LDS, read AHEAD steps before their use: a read takes about
// 128 cycles, a step 32 per product.  (d = 256 in bf16 has registers for two steps: with three, operands, too, are
// reloaded from scratch for every 32 rows; two instead of three took the pass of 3,840 x 1M from 7.17 to 6.73 ms.)  The fences keep the
// compiler from reading further ahead, which would spill the accumulators.
template <int N, int P, typename L, typename M>
__device__ __forceinline__ void pipelined(L&& load, M&& multiply) {
  constexpr int AHEAD = N < 4 ? N - 1 : P == 1 ? (N < 16 ? 3 : 2) : P == 2 ? 2 : 1;
  u32x4 a[AHEAD + 1][P];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) load(i, a[i]);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i + AHEAD < N) load(i + AHEAD, a[(i + AHEAD) % (AHEAD + 1)]);
    multiply(i, a[i % (AHEAD + 1)]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// S += Y X^T of the 32 rows of a tile from `sub`, for NX blocks of X
template <typename G, int NX>
__device__ __forceinline__ void scores(uint32_t tile, int sub, const u32x4 (&x)[NX][G::NS][G::CH / 2],
                                       f32x16 (&s)[NX]) {
  using Q = Products<G::NS>;
  const int lane = threadIdx.x & 63, row = lane & 31;  // 32 more rows leave the swizzle as it is
  const uint32_t base = (tile + (sub * 32 + row) * G::CH * 16) ^ (uint32_t)(swz<G::CH>(row) ^ (lane / 32)) << 4;
  pipelined<G::CH / 2, G::NS>(
      [&](int kk, u32x4(&a)[G::NS]) {
#pragma unroll
        for (int p = 0; p < G::NS; ++p)
          a[p] = lds_read<u32x4>((base ^ (uint32_t)(2 * kk & 15) << 4) + (2 * kk & ~15) * 16 + p * G::PART * 16);
      },
      [&](int kk, const u32x4(&a)[G::NS]) {
#pragma unroll
        for (int q = 0; q < Q::N; ++q)
#pragma unroll
          for (int nb = 0; nb < NX; ++nb) s[nb] = mma<G::HALF>(a[Q::at[q][0]], x[nb][Q::at[q][1]][kk], s[nb]);
      });
}

// the value of the lane with the same X row in the other half
__device__ __forceinline__ float other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// A score in units of log 2.  Beyond fp32's range (|z| > 2.3e38) it is the range's end, so that a row of the type's
// lowest values keeps its order; an infinite score stays one.
__device__ __forceinline__ float in_log2(float s, float k) {
  const float z = s * k;
  return fabsf(s) < INFINITY ? fminf(fmaxf(z, -3.40282347e38f), 3.40282347e38f) : z;
}

// Up to this size of the reference (a maximum or a log-sum, in units of log 2) exponents are taken in one step,
// exp2(s k - reference) with the product not rounded: its distance to the rounded reference is 2^-8 at most.  Beyond it
// (a block of masked items, an outlying row) that distance is no longer small -- 2^75 at 1e30, and exp2 of it infinite --
// so the product is rounded, too, as the reference was.
constexpr float kLarge = 65536.f;

__device__ __forceinline__ float max_or_nan(float a, float b) { return a != a ? a : b != b ? b : fmaxf(a, b); }

// fp32: what a block of 32 rows has been multiplied by, undone: 2^-e of fp16 parts, 1 of bf16 parts, +inf where its
// entries have no such parts (0 behind the last row)
template <typename G>
__device__ __forceinline__ float undo(const float* inv, int64_t row, int64_t rows) {
  if constexpr (G::F32) return row < rows ? inv[row / 32] : 0.f;
  else return 1.f;
}

// the same for the blocks of a tile, block q in lane q; read with undo_of
template <typename G>
__device__ __forceinline__ float undo_tile(const float* inv, int64_t t, int64_t rows) {
  if constexpr (G::F32) return inv[min(t * G::SUBS + (threadIdx.x & 63) % G::SUBS, fr::ceil_div_dev(rows, 32) - 1)];
  else return 1.f;
}
template <typename G>
__device__ __forceinline__ float undo_of(float tile, int sub) {
  if constexpr (G::F32) return lane_value(tile, sub);
  else return 1.f;
}

// Two fp16 parts leave up to 2^-25 of an entry whose block has been brought below 2^14, however small the entry is: of
// a score 2^-10 D k inv_x inv_y in all, in units of log 2, which the limit keeps below 2^-23 (a step of fp32 at 1).
// Blocks beyond it -- an item masked by -1e9, a user row far above the table's -- would spoil the scores of the rows
// beside the outlying one, and are computed from the fp32 rows.  Bf16 parts have fp32's range; there it is only blocks
// with an entry above 2^58, whose products might not add up, or without a finite value.
template <typename G>
constexpr float kPartsLimit = G::HALF ? 0x1p-13f / (G::CH * 8) : 3.40282347e38f;

// S = Y X^T of 32 rows each on the fp32 matrix instruction: an entry's products see that entry alone, infinities and NaN
// are those of the plain formula.  y, x: this lane's rows of d columns, half h taking columns 8 i + 4 h .. + 4; y is
// taken as zero where it is not real.  It waits for its loads (a pass of such blocks alone
// takes 2.6 times as long).
template <int NX>
__device__ __forceinline__ void plain_scores(const float* y, bool real, const float* const (&x)[NX], int d,
                                             f32x16 (&s)[NX]) {
  struct alignas(4) Four {
    float v[4];
  };
#pragma unroll
  for (int nb = 0; nb < NX; ++nb) s[nb] = f32x16{};
#pragma unroll 1
  for (int c = 0; c < d; c += 8) {
    const int at = c + (threadIdx.x & 32) / 8;
    Four a = {}, b[NX] = {};
    if (c + 8 <= d) {
      a = *reinterpret_cast<const Four*>(y + at);
#pragma unroll
      for (int nb = 0; nb < NX; ++nb) b[nb] = *reinterpret_cast<const Four*>(x[nb] + at);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (at + j < d) {
          a.v[j] = y[at + j];
#pragma unroll
          for (int nb = 0; nb < NX; ++nb) b[nb].v[j] = x[nb][at + j];
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int nb = 0; nb < NX; ++nb)
        s[nb] = __builtin_amdgcn_mfma_f32_32x32x2f32(real ? a.v[j] : 0.f, b[nb].v[j], s[nb], 0, 0, 0);
  }
}

// a number that the compiler cannot tell from another: what is computed from it stays where it is used
__device__ __forceinline__ int64_t here(int64_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

// the A operand of the second product: Y columns dt * 32 .. + 32 for the 16 Y rows behind results 8 t .. 8 t + 8
template <int CH>
__device__ __forceinline__ u32x4 columns(uint32_t tile, int sub, int t, int dt) {
  const int lane = threadIdx.x & 63, low = 4 * (lane / 32) + (lane & 15) / 4;
  s16x4 v[2];
#pragma unroll
  for (int jj = 0; jj < 2; ++jj) {
    const int row = 8 * jj + low;                                // 16 more rows leave the swizzle as it is
    const int c = (lane / 16 % 2) * 2 + (lane & 3) / 2;          // of 4 chunks per 32 columns, each read by halves
    // (the half of the chunk before the exclusive or, so that the constants are the reads' own offsets)
    const uint32_t base =
        ((tile + (sub * 32 + row) * CH * 16) ^ (uint32_t)(swz<CH>(row) ^ c) << 4) | (uint32_t)(lane & 1) * 8;
    const uint32_t at = (base ^ (uint32_t)(4 * dt & 15) << 4) + (4 * dt & ~15) * 16 + t * 16 * CH * 16;
    v[jj] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((FR_LDS s16x4*)(uintptr_t)at);
  }
  return __builtin_bit_cast(u32x4, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
}

// 16 results as the second product's operand: per 8 of them NG parts
template <int NG>
__device__ __forceinline__ void operand_of(const f32x16& s, u32x4 (&g)[2][NG]) {
#pragma unroll
  for (int t2 = 0; t2 < 2; ++t2) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = s[8 * t2 + j];
    parts_of<NG>(v, g[t2]);
  }
}

// out^T += Y^T G of the 32 rows of a tile from `sub`
template <typename G, int DT>
__device__ __forceinline__ void accumulate(uint32_t tile, int sub, const u32x4 (&g)[2][G::NG], f32x16 (&acc)[DT]) {
  using Q = Products<G::NG>;
  pipelined<2 * DT, G::NG>(
      [&](int i, u32x4(&y)[G::NG]) {
#pragma unroll
        for (int p = 0; p < G::NG; ++p) y[p] = columns<G::CH>(tile + (G::G0 + p) * G::PART * 16, sub, i / DT, i % DT);
      },
      [&](int i, const u32x4(&y)[G::NG]) {
#pragma unroll
        for (int q = 0; q < Q::N; ++q)
          acc[i % DT] = mma<false>(y[Q::at[q][0]], g[i / DT][Q::at[q][1]], acc[i % DT]);
      });
}

// The workgroup's (row tile, split): neighbouring workgroups of one XCD (block % 8) take the row tiles
// of one split, which stream the same Y rows through that XCD's L2.
__device__ __forceinline__ bool place(int64_t rt_n, int64_t sp_n, int64_t& rt, int64_t& sp) {
  // fewer than 2^32 workgroups (a long division costs half a microsecond)
  const uint32_t b = (uint32_t)fr::block_number(), n = (uint32_t)rt_n;
  const bool eights = sp_n % 8 == 0;
  const uint32_t q = eights ? b / 8 : b, s = q / n;
  sp = eights ? b % 8 + 8 * (int64_t)s : s;
  rt = q - s * n;
  return sp < sp_n;
}

// operands and results in registers, and the workgroups per compute unit that these have to leave room for
template <typename T, int D, bool O>
constexpr int stats_regs(int nx) { return nx * (Geo<T, D, O>::NS * D / 4 + (O ? D / 2 : 0) + 16); }
template <typename T, int D>
constexpr int grad_regs() { return Geo<T, D, true>::NS * D / 4 + D / 2 + 16; }
[[maybe_unused]] constexpr int waves_for(int regs) { return regs > 210 ? 1 : 2; }

// ------------------------------------------------------------------------------ statistics
// Per split and row: the maximum m of the split's scores in units of log 2 (or a bound within 2^8 of it), the sum
// of exp2(z - m) over its items but the target, the target's score (-inf if it is not in the split), and,
// with O, the sum of exp2(z - m) W over its items but the target.
struct StatsArgs {
  const bf16_t *H, *W;  // parts of rows of D columns, part_h / part_w elements apart
  int64_t ldh, part_h, n, ldw, part_w, nv;
  const float *inv_h, *inv_w;
  const float *rows_h, *rows_w;  // fp32: the rows themselves, of d columns
  int64_t ld_rows_h, ld_rows_w;
  int d;
  const int64_t* ids;
  float k;
  int64_t rt_n, sp_n, tiles_per_split;
  float4* stats;  // [split][n]: m, sum, target's score, 0
  float* o;       // [split][n][D]
};

template <typename T, int D, int NX, bool O>
__global__ __launch_bounds__(256, waves_for(stats_regs<T, D, O>(NX))) void stats_kernel(
    StatsArgs a) {
  using G = Geo<T, D, O>;
  constexpr int DT = O ? D / 32 : 1;
  static_assert(!O || NX == 1, "o leaves registers for one block");
  __shared__ alignas(1024) u32x4 tile[2][G::CHUNKS];
  int64_t rt, sp;
  if (!place(a.rt_n, a.sp_n, rt, sp)) return;
  const int lane = threadIdx.x & 63, half = lane / 32, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int64_t x0 = (rt * 4 + wave) * 32 * NX;
  u32x4 x[NX][G::NS][G::CH / 2];
  float kx[NX], m[NX], sum[NX], target[NX];
  int32_t id[NX];
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;
#pragma unroll
  for (int nb = 0; nb < NX; ++nb) {
    const int64_t row = x0 + nb * 32 + (lane & 31);
    load_x<G>(a.H, a.ldh, a.part_h, a.n, x0 + nb * 32, x[nb]);
    kx[nb] = a.k * undo<G>(a.inv_h, x0 + nb * 32, a.n);
    const int64_t t = row < a.n ? a.ids[row] : -1;
    id[nb] = t >= 0 && t < a.nv ? (int32_t)t : -1;
    m[nb] = target[nb] = -INFINITY;
    sum[nb] = 0.f;
  }
  const int64_t t0 = sp * a.tiles_per_split, t1 = min(t0 + a.tiles_per_split, fr::ceil_div_dev(a.nv, G::TY));
  const Stage<G> stage(a.W, a.ldw, a.part_w, a.nv);
  float next = 1.f;
  const auto fetch = [&](int64_t t, int b) {
    stage.load(t, tile[b]);
    next = undo_tile<G>(a.inv_w, t, a.nv);
  };
  if (t0 < t1) fetch(t0, 0);
  for (int64_t t = t0; t < t1; ++t) {
    wait_loads();
    __syncthreads();  // tile t is whole, and the other buffer's readers are done
    const float inv = next;
    if (t + 1 < t1) fetch(t + 1, (int)(t + 1 - t0) & 1);
    const uint32_t cur = lds_of(tile[(t - t0) & 1]);
#pragma unroll 1
    for (int sub = 0; sub < G::SUBS; ++sub) {
      const int y0 = (int)(t * G::TY) + sub * 32, left = (int)min(a.nv - y0, (int64_t)32);
      if (left <= 0) break;
      const float ky = undo_of<G>(inv, sub);
      f32x16 s[NX] = {};
      scores<G, NX>(cur, sub, x, s);
      bool plain = false;
      if constexpr (G::F32) {
#pragma unroll
        for (int nb = 0; nb < NX; ++nb) plain |= !(kx[nb] * ky <= kPartsLimit<G>);
        plain = __ballot(plain);
        if (plain) {
          const float* rows[NX];
#pragma unroll
          for (int nb = 0; nb < NX; ++nb)
            rows[nb] = a.rows_h + here(min(x0 + nb * 32 + (lane & 31), a.n - 1)) * a.ld_rows_h;
          plain_scores<NX>(a.rows_w + here(min(y0 + (lane & 31), (int)a.nv - 1)) * a.ld_rows_w, true, rows, a.d, s);
        }
      }
#pragma unroll
      for (int nb = 0; nb < NX; ++nb) {
        // tiny rows' scales may underflow together: not to 0, which times a masked -inf would be NaN
        float k = plain ? a.k : G::HALF ? fmaxf(kx[nb] * ky, 1.17549435e-38f) : kx[nb] * ky;
        if (left < 32) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (result_row(r, 0) >= left - 4 * half) s[nb][r] = -INFINITY;
        }
        const int at = id[nb] - y0;  // the target among the tile's rows
        if (__ballot(at >= 0 && at < 32)) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (result_row(r, 0) == at - 4 * half) {
              target[nb] = in_log2(s[nb][r], k);
              s[nb][r] = -INFINITY;
            }
        }
        float top = s[nb][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, s[nb][r]);
        top = in_log2(top, k);
        if constexpr (O) {
          top = fmaxf(top, other_half(top));  // both halves' results meet in one product: one maximum
          if (__ballot(top > m[nb] + 8.f)) {
            const float m_new = fmaxf(m[nb], top), keep = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[nb] - m_new);
            m[nb] = m_new;
            sum[nb] *= keep;
            // (what weighs nothing is dropped: items masked by the type's lowest value may have summed up to -inf)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int r = 0; r < 16; ++r) acc[dt][r] = keep == 0.f ? 0.f : acc[dt][r] * keep;
          }
        } else {
          const float m_new = fmaxf(m[nb], top);
          sum[nb] *= m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[nb] - m_new);
          m[nb] = m_new;
        }
        float base = m[nb] == -INFINITY ? 0.f : m[nb];  // nothing seen yet: exp2(-inf - 0) = 0
        if (__ballot(!(fabsf(base) <= kLarge))) {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[nb][r] = in_log2(s[nb][r], k) - base;
          k = 1.f;
          base = 0.f;
        }
        float e = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[nb][r], k, -base));
          if constexpr (O) s[nb][r] = p;
          e += p;
        }
        sum[nb] += e;
      }
      if constexpr (O) {
        u32x4 g[2][G::NG];
        operand_of(s[0], g);
        accumulate<G, DT>(cur, sub, g, acc);
      }
    }
  }
#pragma unroll
  for (int nb = 0; nb < NX; ++nb) {
    const int64_t row = x0 + nb * 32 + (lane & 31);
    const float mm = fmaxf(m[nb], other_half(m[nb]));
    const float mine = sum[nb] == 0.f ? 0.f : sum[nb] * __builtin_amdgcn_exp2f(m[nb] - mm);  // a NaN stays one
    const float both = mine + other_half(mine), z = max_or_nan(target[nb], other_half(target[nb]));
    if (row >= a.n) continue;
    if (lane < 32) a.stats[sp * a.n + row] = make_float4(mm, both, z, 0.f);
    if constexpr (O) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4*>(a.o + (sp * a.n + row) * D + dt * 32 + 8 * q + 4 * half) =
              f32x4{acc[dt][4 * q], acc[dt][4 * q + 1], acc[dt][4 * q + 2], acc[dt][4 * q + 3]};
    }
  }
}

// The splits' statistics joined in their order, logp, lse (log 2 units, as a score and the logarithm of the sum beside
// it: in one number the score could swallow the logarithm) and, with O, o and 1 - p of the target.
// A group of D / 4 lanes per row, or (WIDE, for few rows of many splits) a workgroup per row, whose groups take
// the splits in turn and are joined in group order.
struct FinishArgs {
  const float4* stats;
  const float* part;
  int64_t sp_n, n, nv;
  const int64_t* ids;
  int d;
  float *logp, *lse2, *o, *rest;
};

template <int D, bool O, bool WIDE>
__global__ __launch_bounds__(WIDE ? 1024 : 256) void finish_kernel(FinishArgs a) {
  constexpr int L = D / 4, NG = WIDE ? 1024 / L : 1, PER = L * NG;  // threads per row
  __shared__ float red[WIDE ? 48 : 1];
  __shared__ f32x4 red_o[O && WIDE ? NG : 1][O && WIDE ? L : 1];
  __shared__ float red_s[O && WIDE ? NG : 1];
  const int64_t row = WIDE ? fr::block_number() : fr::block_number() * (256 / L) + threadIdx.x / L;
  const int t = threadIdx.x % PER, g = t / L, wave = threadIdx.x / 64;
  if (row >= a.n) return;
  const int64_t id = a.ids[row];
  const bool real = id >= 0 && id < a.nv;
  float m = -INFINITY, z = -INFINITY;
  for (int64_t q = t; q < a.sp_n; q += PER) {
    const float4 v = a.stats[q * a.n + row];
    m = fmaxf(m, v.x);
    z = max_or_nan(z, v.z);
  }
  constexpr int S = PER < 64 ? PER : 64;
#pragma unroll
  for (int off = S / 2; off > 0; off >>= 1) {
    m = fmaxf(m, __shfl_xor(m, off, S));
    z = max_or_nan(z, __shfl_xor(z, off, S));
  }
  if constexpr (WIDE) {
    if ((threadIdx.x & 63) == 0) {
      red[wave] = m;
      red[16 + wave] = z;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      m = fmaxf(m, red[i]);
      z = max_or_nan(z, red[16 + i]);
    }
  }
  const float base = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if constexpr (O) {
#pragma unroll 4
    for (int64_t q = g; q < a.sp_n; q += NG) {
      const float4 v = a.stats[q * a.n + row];
      const float w = __builtin_amdgcn_exp2f(v.x - base);
      sum = fmaf(v.y, w, sum);
      const f32x4 part = *reinterpret_cast<const f32x4*>(a.part + (q * a.n + row) * D + t % L * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = w == 0.f ? o[j] : fmaf(part[j], w, o[j]);
    }
    if constexpr (WIDE) {
      red_o[g][t % L] = o;
      if (t % L == 0) red_s[g] = sum;
      __syncthreads();
      if (g) return;
      o = red_o[0][t];
      sum = red_s[0];
      for (int i = 1; i < NG; ++i) {
        o += red_o[i][t];
        sum += red_s[i];
      }
    }
  } else {
    for (int64_t q = t; q < a.sp_n; q += PER) {
      const float4 v = a.stats[q * a.n + row];
      sum = fmaf(v.y, __builtin_amdgcn_exp2f(v.x - base), sum);
    }
    sum = group_sum<S>(sum);
    if constexpr (WIDE) {
      if ((threadIdx.x & 63) == 0) red[32 + wave] = sum;
      __syncthreads();
      sum = red[32];
#pragma unroll
      for (int i = 1; i < 16; ++i) sum += red[32 + i];
    }
  }
  // the larger of the others' maximum and the target's score as the reference
  const float top = fmaxf(m, z), low = top == -INFINITY ? 0.f : top;
  const float share = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - low);  // no other items: sum is 0 (or NaN)
  const float others = sum * share, total = others + __builtin_amdgcn_exp2f(z - low);
  const float l2 = __builtin_log2f(total);
  if constexpr (O) {
    const float w = share / total;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (t * 4 + j < a.d) a.o[row * a.d + t * 4 + j] = o[j] * w;
  }
  if (t) return;
  if (a.lse2) {
    a.lse2[row] = low;
    a.lse2[a.n + row] = l2;
  }
  if (a.rest) a.rest[row] = others / total;
  // (an infinite score is no reference: NaN where it is +inf, or where the row has nothing but -inf)
  const float lp = z >= m && fabsf(z) < INFINITY ? -log1pf(others) : ((z - low) - l2) * 0.6931471805599453f;
  a.logp[row] = !real ? 0.f : lp >= 0.f ? -0.f : lp;  // +0 is the mark of a row without a target
}

// dH[row, :d] = a c ((1 - p) W[target] - o): zeros without a target
template <typename T>
__global__ __launch_bounds__(256) void dh_kernel(const float* __restrict__ o, const float* __restrict__ rest,
                                                 const float* __restrict__ up, float c, const T* __restrict__ W,
                                                 int64_t ldw, int64_t nv, const int64_t* __restrict__ ids, int64_t n,
                                                 int d, T* __restrict__ dh) {
  const int64_t e = fr::block_number() * 256 + threadIdx.x;
  if (e >= n * d) return;
  const int64_t row = e / d;
  const int64_t id = ids[row];
  const float a = up[row] * c;
  float v = 0.f;
  if (id >= 0 && id < nv && a != 0.f) v = a * fmaf(rest[row], fr::to_f32(W[id * ldw + e % d]), -o[e]);
  dh[e] = fr::from_f32<T>(v);
}

// ------------------------------------------------------------------------------- operands
// Rows as the kernels take them: parts of D columns, zeros behind the d-th.  With ids: a row without a target
// (padding) is zero throughout, so that whatever it holds spreads neither into dW nor into the scale of the
// rows around it.  For the gradients' users also, per row up to n_out: lse in one number (+inf without a target: its
// probabilities are 0; for bf16 -lse / (c log2 e), which the products are added to), the coefficient a_n c, the
// target and its entry a_n c (1 - p); and inv is negative where one of the 32 has an lse beyond kLarge (or too large
// for fp32 in the scores' units; the block's lse are then 0 here), for bf16 1/2 where one has no target.
template <typename T>
struct Rows {
  const T* src;  // null: no rows
  int64_t ld, n, n_out;
  bool vec;
  bf16_t* out;  // [part][n_out][D]
  float* inv;   // per 32 rows 2^-e of fp16 parts, else 1 (and see above)
  const int64_t* ids;
  int64_t nv;
  const float *lse2, *rest, *up;
  float c;
  float *lse_o, *coef, *target;  // null: no statistics
  int32_t* ids_o;
};

// 32 rows per group of threads: TG of them, K chunks of eight columns each
template <typename T, int D, bool GRAD>
__global__ __launch_bounds__(256) void rows_kernel(Rows<T> h, Rows<T> w, int d) {
  using G = Geo<T, D, GRAD>;
  constexpr int TG = D >= 64 ? 256 : 128, K = 32 * G::CH / TG;
  __shared__ uint32_t red[4], red_kind[4];
  const int64_t gh = h.src ? fr::ceil_div_dev(h.n_out, 32) : 0;
  const int64_t block = fr::block_number() * (256 / TG) + threadIdx.x / TG;
  const bool users = block < gh;
  const Rows<T>& a = users ? h : w;
  const int64_t g = users ? block : block - gh;
  float v[K][8];
  uint32_t top = 0;
  uint32_t kind = 0;  // 1: a user without a target, 2: one of a large lse, 4: an entry that is no number
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int q = k * TG + threadIdx.x % TG, col = q % G::CH * 8;
    const int64_t row = g * 32 + q / G::CH;
    const int64_t id = a.ids && row < a.n ? a.ids[row] : 0;
    const bool real = a.src && row < a.n && (!a.ids || (id >= 0 && id < a.nv));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[k][j] = 0.f;
    if (real) {
      const T* x = a.src + row * a.ld + col;
      if (a.vec) {
#pragma unroll
        for (int j = 0; j < 8; j += fr::kVec<T>) fr::Vec<T, fr::kVec<T>>::load(x + j, v[k] + j);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (col + j < d) v[k][j] = fr::to_f32(x[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t u = __float_as_uint(v[k][j]) & 0x7fffffffu;
      if (u < 0x7f800000u) top = max(top, u);  // the largest finite entry
      else kind |= 4u;
    }
    if (a.coef && col == 0 && row < a.n_out) {
      const float lse = real ? a.lse2[row] + a.lse2[a.n + row] : INFINITY;
      const float start = G::F32 ? lse : real ? lse / (a.c * -kLog2e) : -INFINITY;
      kind |= !real ? 1u : fabsf(lse) <= kLarge && fabsf(start) < INFINITY ? 0u : 2u;
      a.lse_o[row] = start;
      a.coef[row] = real ? a.up[row] * a.c : 0.f;
      a.target[row] = real ? a.up[row] * a.c * a.rest[row] : 0.f;
      a.ids_o[row] = real ? (int32_t)id : -1;
    }
  }
  float scale = 1.f, undo = 1.f;
  if constexpr (G::F32 || GRAD) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
      kind |= (uint32_t)__shfl_xor((int)kind, off, 64);
    }
    if ((threadIdx.x & 63) == 0) {
      red[threadIdx.x / 64] = top;
      red_kind[threadIdx.x / 64] = kind;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TG / 64; ++i) {
      top = max(top, red[threadIdx.x / TG * (TG / 64) + i]);
      kind |= red_kind[threadIdx.x / TG * (TG / 64) + i];
    }
    if constexpr (G::HALF) {
      const int e = min(13 - ((int)(top >> 23) - 127), 120);  // largest in [2^13, 2^14), 2^e finite
      scale = __uint_as_float((uint32_t)(e + 127) << 23);
      undo = __uint_as_float((uint32_t)(127 - e) << 23);
    }
    if (kind & 2) {  // the kernel takes these users' lse from the forward's two numbers
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int q = k * TG + threadIdx.x % TG;
        const int64_t row = g * 32 + q / G::CH;
        if (q % G::CH == 0 && row < a.n && a.ids_o[row] >= 0) a.lse_o[row] = 0.f;
      }
    }
    if (G::F32 && (kind & 4 || (!G::HALF && top > 0x5c800000u /* 2^58 */))) undo = INFINITY;
    if (a.src && threadIdx.x % TG == 0 && g * 32 < a.n_out)
      a.inv[g] = kind & 2 ? -undo : !G::F32 && kind & 1 ? 0.5f : undo;
  }
  if (!a.src) return;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int q = k * TG + threadIdx.x % TG;
    const int64_t row = g * 32 + q / G::CH;
    if (row >= a.n_out) continue;
    bf16_t* out = a.out + row * D + q % G::CH * 8;
    const int64_t part = a.n_out * D;
    if constexpr (G::HALF) {
      u32x4 o[2];
      halves_of(v[k], scale, o);
      *reinterpret_cast<u32x4*>(out) = o[0];
      *reinterpret_cast<u32x4*>(out + part) = o[1];
    }
    if constexpr (GRAD || !G::HALF) {
      u32x4 o[G::NG];
      row_parts_of<G::NG>(v[k], o);
#pragma unroll
      for (int p = 0; p < G::NG; ++p) *reinterpret_cast<u32x4*>(out + (G::G0 + p) * part) = o[p];
    }
  }
}

// ------------------------------------------------------------------------------- gradients
struct GradArgs {
  const bf16_t *X, *Y;  // rows of D columns, their parts part_x / part_y elements apart
  int64_t ldx, part_x, nx, ldy, part_y, ny;
  const float *inv_x, *inv_y;
  const float *rows_x, *rows_y;  // fp32: the rows themselves, of d columns (users: the n that are there)
  int64_t ld_rows_x, ld_rows_y, n;
  const float *lse, *coef, *target;  // per user, to a multiple of TY rows, plus 64
  const int32_t* ids;
  const float *lse2, *lse2_sum;  // the forward's, [n] each
  float k;
  int64_t rt_n, sp_n, tiles_per_split;
  float* part;  // [split][nx][D], or null: one split, rows written to out
  void* out;
  int64_t ldo;
  int d;
};

// dW: X = items, Y = users
template <typename T, int D>
__global__ __launch_bounds__(256, waves_for(grad_regs<T, D>())) void grad_kernel(GradArgs a) {
  using G = Geo<T, D, true>;
  constexpr int DT = D / 32;
  constexpr int UR = G::TY < 64 ? 64 : G::TY;  // user values per tile: whole waves of 64
  __shared__ alignas(1024) u32x4 tile[2][G::CHUNKS];
  __shared__ alignas(16) float u_lse[2][UR], u_coef[2][UR], u_target[2][UR];
  __shared__ alignas(16) int32_t u_id[2][UR];
  int64_t rt, sp;
  if (!place(a.rt_n, a.sp_n, rt, sp)) return;
  const int lane = threadIdx.x & 63, half = lane / 32, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int64_t x0 = (rt * 4 + wave) * 32, xl = x0 + (lane & 31);
  u32x4 x[1][G::NS][G::CH / 2];
  load_x<G>(a.X, a.ldx, a.part_x, a.nx, x0, x[0]);
  const float kx = a.k * undo<G>(a.inv_x, x0, a.nx);
  // An infinite or NaN entry among the wave's items makes NaN of a zero row's score, so that blocks of users some of
  // whom have no target (inv = 1/2) take the slower way, too.
  const float slow = !G::F32 && has_no_number(x[0]) ? 1.f : 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;

  const Stage<G> stage(a.Y, a.ldy, a.part_y, a.ny);
  float next = 1.f;
  const auto fetch = [&](int64_t t, int b, bool flags) {
    if (flags) next = a.inv_y[t * G::SUBS + (threadIdx.x & 63) % G::SUBS];  // block q of the tile in lane q
    stage.load(t, tile[b]);
#pragma unroll
    for (int q = 0; q < UR / 64; ++q) {
      const int64_t u = t * G::TY + q * 64 + lane;
      if (wave == 0)
        __builtin_amdgcn_global_load_lds((const FR_GLOBAL void*)(a.lse + u), (FR_LDS void*)(u_lse[b] + q * 64), 4, 0, 0);
      if (wave == 1)
        __builtin_amdgcn_global_load_lds((const FR_GLOBAL void*)(a.coef + u), (FR_LDS void*)(u_coef[b] + q * 64), 4, 0, 0);
      if (wave == 2)
        __builtin_amdgcn_global_load_lds((const FR_GLOBAL void*)(a.ids + u), (FR_LDS void*)(u_id[b] + q * 64), 4, 0, 0);
      if (wave == 3)
        __builtin_amdgcn_global_load_lds((const FR_GLOBAL void*)(a.target + u), (FR_LDS void*)(u_target[b] + q * 64), 4, 0,
                                         0);
    }
  };

  const int64_t t0 = sp * a.tiles_per_split, t1 = min(t0 + a.tiles_per_split, fr::ceil_div_dev(a.ny, G::TY));
  const auto run = [&](auto f) {
    constexpr bool FLAGS = decltype(f)::value;  // blocks of users are looked at one by one
    if (t0 < t1) fetch(t0, 0, FLAGS);
    for (int64_t t = t0; t < t1; ++t) {
      wait_loads();
      __syncthreads();
      const float inv = next;
      if (t + 1 < t1) fetch(t + 1, (int)(t + 1 - t0) & 1, FLAGS);
      const int b = (int)(t - t0) & 1;
      const uint32_t cur = lds_of(tile[b]);
  #pragma unroll 1
      for (int sub = 0; sub < G::SUBS; ++sub) {
        if (t * G::TY + sub * 32 >= a.ny) break;
        const float ky = FLAGS ? lane_value(inv, sub) : 1.f;
        float k = G::F32 ? kx * fabsf(ky) : a.k;
        const bool plain = G::F32 && __ballot(!(k <= kPartsLimit<G>));
        const bool large = FLAGS && (ky < slow || plain);  // negative: users whose lse is too large for one number
        if constexpr (G::HALF) k = fmaxf(k, 1.17549435e-38f);
        f32x16 s[1] = {};
        if constexpr (!G::F32) {  // the products are added to -lse / k: their roundings at its size are below p's to bf16
  #pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 l = *reinterpret_cast<const f32x4*>(&u_lse[b][sub * 32 + 8 * q + 4 * half]);
  #pragma unroll
            for (int j = 0; j < 4; ++j) s[0][4 * q + j] = l[j];
          }
        }
        const int32_t uid = u_id[b][sub * 32 + (lane & 31)];
        scores<G, 1>(cur, sub, x, s);
        if (plain) {
          const float* const rows[1] = {a.rows_x + here(min(xl, a.nx - 1)) * a.ld_rows_x};
          const int64_t y = here(min(t * G::TY + sub * 32 + (lane & 31), a.n - 1));
          plain_scores<1>(a.rows_y + y * a.ld_rows_y, uid >= 0, rows, a.d, s);
          k = a.k;
        }
        const bool hit = __ballot((uint32_t)uid - (uint32_t)x0 < 32u);  // a target of the tile is among the wave's items
        if (large) {  // the exponents themselves, of users with an item (which are among the forward's n rows)
  #pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int u = sub * 32 + result_row(r, half);
            float e = -INFINITY;
            if (u_id[b][u] >= 0) {
              const uint32_t at = (uint32_t)(t * G::TY) + u;
              e = in_log2(s[0][r], k);
              if (ky < 0.f) e = (e - a.lse2[at]) - a.lse2_sum[at];
            }
            s[0][r] = e;
            __builtin_amdgcn_sched_barrier(0);  // a few values at a time
          }
          k = 1.f;
        }
  #pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x4 l = {0.f, 0.f, 0.f, 0.f};
          if constexpr (G::F32) l = *reinterpret_cast<const f32x4*>(&u_lse[b][sub * 32 + 8 * q + 4 * half]);
          const f32x4 c = *reinterpret_cast<const f32x4*>(&u_coef[b][sub * 32 + 8 * q + 4 * half]);
  #pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = __builtin_amdgcn_exp2f(G::F32 ? fmaf(s[0][4 * q + j], k, -l[j]) : s[0][4 * q + j] * k);
            s[0][4 * q + j] = -c[j] * p;
          }
        }
        // the target's entry is a_n c (1 - p), from the forward's 1 - p
        const auto targets = [&](auto&& put) {
  #pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(&u_target[b][sub * 32 + 8 * q + 4 * half]);
            const int4 id = *reinterpret_cast<const int4*>(&u_id[b][sub * 32 + 8 * q + 4 * half]);
            put(4 * q, id.x == (int)xl, v[0]);
            put(4 * q + 1, id.y == (int)xl, v[1]);
            put(4 * q + 2, id.z == (int)xl, v[2]);
            put(4 * q + 3, id.w == (int)xl, v[3]);
            __builtin_amdgcn_sched_barrier(0);  // a few values at a time
          }
        };
        if (hit) targets([&](int r, bool at, float v) { s[0][r] = at ? v : s[0][r]; });
        u32x4 g[2][G::NG];
        operand_of(s[0], g);
        // bf16: what is left of the targets' entries in a second pass (the same code: the registers of one).  Without
        // it dW is off by 0.0024-0.0025 of its norm, of few users by up to 0.004, with it by 0.0017, its own rounding;
        // it costs nothing in 3,840 x 1M x 256 (6.7 ms) and 13-21 % of the pass where blocks of items are hit often
        // (7,168 x 45,630 x 64 256 -> 309 us, 4,200 x 60,000 x 128 320 -> 385, 1,000 x 60,000 x 64 82 -> 97).
        const int passes = hit && !G::F32 ? 2 : 1;
  #pragma unroll 1
        for (int pass = 0; pass < passes; ++pass) {
          if (pass) {
            f32x16 r16;
            targets([&](int r, bool at, float v) { r16[r] = at ? v - fr::to_f32(fr::from_f32<bf16_t>(v)) : 0.f; });
            operand_of(r16, g);
          }
          accumulate<G, DT>(cur, sub, g, acc);
        }
      }
    }
  };
  if constexpr (D < 256) {
    run(std::true_type{});
  } else {
    // a loop of its own where none of the workgroup's blocks needs them (3,840 x 1M x 256 bf16 3.3 ms, 3.6 with the flags
    // read and tested per tile; narrower ones have the registers)
    static_assert(!G::HALF);
    bool any = false;
    for (int64_t i = t0 * G::SUBS + threadIdx.x; i < min(t1 * G::SUBS, a.ny / 32); i += 256)
      any |= a.inv_y[i] < slow || !(kx * a.inv_y[i] <= kPartsLimit<G>);
    if (__syncthreads_or(any)) run(std::true_type{});
    else run(std::false_type{});
  }
  if (xl >= a.nx) return;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int col = dt * 32 + 8 * q + 4 * half;
      const f32x4 v = {acc[dt][4 * q], acc[dt][4 * q + 1], acc[dt][4 * q + 2], acc[dt][4 * q + 3]};
      if (a.part) {
        *reinterpret_cast<f32x4*>(a.part + (sp * a.nx + xl) * D + col) = v;
      } else {
        T* o = static_cast<T*>(a.out) + xl * a.ldo + col;
        if (a.d == D) {  // contiguous rows of D: four columns at a time
          if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(o) = v;
          else *reinterpret_cast<uint2*>(o) = make_uint2(fr::pack_bf16(v[0], v[1]), fr::pack_bf16(v[2], v[3]));
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (col + j < a.d) o[j] = fr::from_f32<T>(v[j]);
        }
      }
    }
}

// dW[x, :d] = sum over splits of part[split][x][:], in split order
template <typename T, int D>
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ part, int64_t sp_n, int64_t rows,
                                                   T* __restrict__ out, int d) {
  const int64_t e = fr::block_number() * 256 + threadIdx.x;
  if (e >= rows * (D / 4)) return;
  const int64_t row = e / (D / 4);
  const int col = (int)(e % (D / 4)) * 4;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int64_t q = 0; q < sp_n; ++q) s += *reinterpret_cast<const f32x4*>(part + (q * rows + row) * D + col);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (col + j < d) out[row * d + col + j] = fr::from_f32<T>(s[j]);
}

// --------------------------------------------------------------------------- preference loss
// A position without a target (item_logp_fwd's +0; a target's value is -0 or less) has no log ratio: whatever the
// reference holds there takes no part.
__device__ __forceinline__ bool lost(float logp, const float* ref) { return ref && __float_as_uint(logp) == 0u; }

// One wave per pair: its margin, its share of the loss (returned), and the gradient of every list member's
// logp for a unit upstream gradient (a list's members share it).
__device__ __forceinline__ float pair_loss_of(const float* __restrict__ logp, const float* __restrict__ ref,
                                              const int64_t* __restrict__ off, int64_t pairs, int64_t p, int64_t n,
                                              float beta, float smooth, float* __restrict__ grad) {
  const int lane = threadIdx.x & 63;
  int64_t lo[2], hi[2];
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    lo[k] = min(max(off[p + k * pairs], (int64_t)0), n);
    hi[k] = min(max(off[p + k * pairs + 1], lo[k]), n);
    double v = 0.0;
    for (int64_t i = lo[k] + lane; i < hi[k]; i += 64)
      if (!lost(logp[i], ref)) v += (double)logp[i] - (ref ? (double)ref[i] : 0.0);
    s += k ? -v : v;
  }
  s = group_sum_d<64>(s);
  const float m = (float)((double)beta * s);
  const float e = expf(-fabsf(m)), down = 1.f / (1.f + e), up = e / (1.f + e);  // sigma(|m|), sigma(-|m|)
  const float sig = m >= 0.f ? down : up, sig_neg = m >= 0.f ? up : down;
  const float tail = log1pf(e);
  const float g = beta / (float)pairs * (smooth * sig - (1.f - smooth) * sig_neg);
#pragma unroll
  for (int k = 0; k < 2; ++k)
    for (int64_t i = lo[k] + lane; i < hi[k]; i += 64) grad[i] = lost(logp[i], ref) ? 0.f : k ? -g : g;
  const float loss = (1.f - smooth) * (fmaxf(-m, 0.f) + tail);
  return smooth > 0.f ? loss + smooth * (fmaxf(m, 0.f) + tail) : loss;  // not 0 times an infinite margin
}

// Few pairs: everything in one workgroup, the clearing of the gradient and the mean included
constexpr int64_t kFewPairs = 64, kFewPositions = 1 << 14;

__global__ __launch_bounds__(1024) void pairs_few_kernel(const float* __restrict__ logp, const float* __restrict__ ref,
                                                         const int64_t* __restrict__ off, int64_t pairs, int64_t n,
                                                         float beta, float smooth, float* __restrict__ loss,
                                                         float* __restrict__ grad) {
  __shared__ double red[16];
  for (int64_t i = threadIdx.x; i < n; i += 1024) grad[i] = 0.f;
  __syncthreads();
  double s = 0.0;
  for (int64_t p = threadIdx.x / 64; p < pairs; p += 16) s += (double)pair_loss_of(logp, ref, off, pairs, p, n, beta, smooth, grad);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x / 64] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = red[0];
    for (int i = 1; i < 16; ++i) s += red[i];
    *loss = (float)(s / (double)pairs);
  }
}

__global__ __launch_bounds__(256) void clear_kernel(float* __restrict__ p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0.f;
}

__global__ __launch_bounds__(256) void pair_kernel(const float* __restrict__ logp, const float* __restrict__ ref,
                                                   const int64_t* __restrict__ off, int64_t pairs, int64_t n,
                                                   float beta, float smooth, float* __restrict__ pair_loss,
                                                   float* __restrict__ grad) {
  const int64_t p = fr::block_number() * 4 + threadIdx.x / 64;
  if (p >= pairs) return;
  const float l = pair_loss_of(logp, ref, off, pairs, p, n, beta, smooth, grad);
  if ((threadIdx.x & 63) == 0) pair_loss[p] = l;
}

__global__ __launch_bounds__(1024) void pair_mean_kernel(const float* __restrict__ pair_loss, int64_t pairs,
                                                         float* __restrict__ loss) {
  __shared__ double red[16];
  double s = 0.0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < pairs; i += 1024) s += (double)pair_loss[i];
  s = group_sum_d<64>(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x / 64] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = red[0];
    for (int i = 1; i < 16; ++i) s += red[i];
    *loss = (float)(s / (double)pairs);
  }
}

// ---------------------------------------------------------------------------------------- host
struct Split {
  int64_t rt, sp, per;  // row tiles, splits, Y tiles per split
  int64_t blocks() const { return sp % 8 == 0 ? 8 * rt * (sp / 8) : rt * sp; }
};

// Splits of the long axis: the number that is estimated to cost the least time.  `tile` is a tile's time on a unit
// that is kept busy; one, two and three workgroups on a unit leave it idle for a part of that (kIdle), and `res`
// find room at a time.  From eight splits on they come in eights, one per XCD of 32 units (see place()).  Every
// round of workgroups costs kExtra for its operands and results, every split one more partial's writing and
// reading at the rate of a copy.
// 1,800 x 29,943 x 128 bf16, us: 48 splits 36, 64 31, 72 35, 96 30, 128 32; 3,840 x 1M x 256 bf16 with o, ms with the
// joining (tiles' addresses computed anew each time): 128 splits 3.74, 64 3.84, 72 3.88, 8 5.15; the pass of 4,200 x
// 60,000 x 128 bf16, us by the splits of dW: 1 403, 3 378, 8 413.
constexpr double kExtra = 3e-6, kIdle[3] = {1.6, 1.2, 1.02}, kCopyRate = 4.7e12;
// a unit's product rate, and the vector work per score beside it (exponential, maximum, sum)
constexpr double kProductRate = 1.3e15 / 256, kScore = 2.5e-11;
constexpr int64_t kMaxSplits = 512;
// From kWideSplits splits and up to kWideRows rows a workgroup joins each row's splits instead of a group of lanes
// (us, group / workgroup): 8 rows, 33,037 x 200 fp32 37 / 11; 80 rows, 43,195 x 128 bf16 28 / 8; 500 rows,
// 60,000 x 256 bf16 16.7 / 14.6; 1,000 rows 12.1 / 16.9, with d = 32 11.7 / 28; 224 rows, 1,500 x 64 fp32 (47 splits)
// 5.6 / 6.6.
constexpr int64_t kWideSplits = 64, kWideRows = 256;

Split split_of(int64_t rows, int64_t rows_per_wg, int64_t tiles, double tile, int res, double split_bytes) {
  Split best{};
  const int64_t rt = fr::ceil_div(rows, rows_per_wg);
  const auto shared = [](int64_t m) { return m > 0 ? (double)m * (m <= 3 ? kIdle[m - 1] : 1.0) : 0.0; };
  double least = INFINITY;
  for (int64_t sp = 1; sp <= std::min(tiles, kMaxSplits); sp += sp < 8 ? 1 : 8) {
    const int64_t per = fr::ceil_div(tiles, sp), used = fr::ceil_div(tiles, per);
    const bool eights = sp % 8 == 0;
    const int64_t wgs = eights ? rt * fr::ceil_div(used, 8) : rt * used, units = eights ? 32 : 256;
    const int64_t full = wgs / (units * res), left = fr::ceil_div(wgs - full * units * res, units);
    const double cost = (double)per * tile * ((double)full * shared(res) + shared(left)) +
                        (double)(full + (left > 0)) * kExtra + (sp > 1 ? (double)sp * split_bytes / kCopyRate : 0.0);
    if (cost < least) {
      least = cost;
      best = Split{rt, sp, per};
    }
  }
  return best;
}

bool shape_ok(int64_t n, int64_t nv, int d) {
  return n >= 0 && n < ((int64_t)1 << 31) && nv >= 1 && nv < ((int64_t)1 << 31) - 64 && d >= 1 && d <= kMaxD;
}

// a unit's time for a workgroup's rows and a tile
constexpr double tile_time(int rows, int tile, int D, int products) {
  return (2.0 * D * products / kProductRate + kScore) * rows * tile;
}

// workgroups that find room on a unit: operands in registers and some 56 more of 512, two tiles in LDS
constexpr int resident(int regs, int chunks) {
  const int by_regs = 512 / (regs + 56), by_lds = 163840 / (2 * chunks * 16 + 4096);
  const int r = by_regs > waves_for(regs) ? by_regs : waves_for(regs);
  return r < by_lds ? r : by_lds;
}

// rows can be taken as they are: bf16 of full width, 16-byte aligned, a tile of them within 32-bit offsets
template <typename T>
bool direct(int d, int D, int64_t ld) {
  return sizeof(T) == 2 && d == D && ld % 8 == 0 && ld < ((int64_t)1 << 22);
}

struct Carver {
  char* base;
  int64_t at = 0;
  template <typename P>
  P* take(int64_t count) {
    P* p = reinterpret_cast<P*>(base + at);
    at += fr::align_up(std::max<int64_t>(count, 1) * (int64_t)sizeof(P), 256);
    return p;
  }
};

// Blocks of 32 users per wave in the statistics: two halve the LDS reads per product, one leaves registers for more
// workgroups per unit.  us, one / two: statistics alone 3,840 x 500,000 x 256 bf16 925 / 813, 7,168 x 45,630 x 64 fp32 153 /
// 146; passes with gradients (o and dW both with one / two) 7,168 x 45,630 x 64 bf16 303 / 352, 1,000 x 60,000 x 64
// 106 / 127.  In fp32 with d = 256 two do not fit.
template <typename T, int D, bool O>
constexpr int stats_blocks() { return O || (sizeof(T) == 4 && D == 256) ? 1 : 2; }

struct FwdWS {
  float4* stats;
  float *o, *inv_h, *inv_w;
  bf16_t *h, *w;  // parts of the users and of the table, where needed
  Split sp;
  int nx;
  int64_t bytes;
};

template <typename T, int D, bool O>
FwdWS fwd_ws(void* base, int64_t n, int64_t nv, int d, int64_t ldw) {
  using G = Geo<T, D, O>;
  FwdWS w;
  w.nx = n > 128 ? stats_blocks<T, D, O>() : 1;
  w.sp = split_of(std::max<int64_t>(n, 1), 128 * w.nx, fr::ceil_div(nv, G::TY),
                  tile_time(128 * w.nx, G::TY, D, Products<G::NS>::N + (O ? Products<G::NG>::N : 0)),
                  resident(stats_regs<T, D, O>(w.nx), G::CHUNKS),
                  (O ? 8.0 * D : 32.0) * n);
  Carver c{static_cast<char*>(base)};
  w.stats = c.take<float4>(w.sp.sp * n);
  w.o = c.take<float>(O ? w.sp.sp * n * D : 1);
  w.h = c.take<bf16_t>(n * D * G::P);
  w.w = c.take<bf16_t>(direct<T>(d, D, ldw) ? 1 : nv * D * G::P);
  w.inv_h = c.take<float>(fr::ceil_div(n, 32));
  w.inv_w = c.take<float>(fr::ceil_div(nv, 32));
  w.bytes = c.at;
  return w;
}

struct BwdWS {
  bf16_t *hs, *w;
  float *inv_h, *inv_w, *lse, *coef, *target, *part;
  int32_t* ids;
  Split v;
  int64_t n_pad, bytes;
};

template <typename T, int D>
BwdWS bwd_ws(void* base, int64_t n, int64_t nv, int d, int64_t ldw) {
  using G = Geo<T, D, true>;
  BwdWS w;
  w.n_pad = fr::align_up(std::max<int64_t>(n, 1), G::TY);  // whole LDS tiles
  w.v = split_of(nv, 128, fr::ceil_div(w.n_pad, G::TY),
                 tile_time(128, G::TY, D, Products<G::NS>::N + Products<G::NG>::N),
                 resident(grad_regs<T, D>(), G::CHUNKS), 8.0 * nv * D);
  Carver c{static_cast<char*>(base)};
  w.hs = c.take<bf16_t>(w.n_pad * D * G::P);
  w.lse = c.take<float>(w.n_pad + 64);
  w.coef = c.take<float>(w.n_pad + 64);
  w.target = c.take<float>(w.n_pad + 64);
  w.ids = c.take<int32_t>(w.n_pad + 64);
  w.w = c.take<bf16_t>(direct<T>(d, D, ldw) ? 1 : nv * D * G::P);
  w.inv_h = c.take<float>(w.n_pad / 32);
  w.inv_w = c.take<float>(fr::ceil_div(nv, 32));
  w.part = c.take<float>(w.v.sp > 1 ? w.v.sp * nv * D : 1);
  w.bytes = c.at;
  return w;
}

template <typename F>
auto by_width(int d, F&& f) {
  if (d <= 32) return f(std::integral_constant<int, 32>{});
  if (d <= 64) return f(std::integral_constant<int, 64>{});
  if (d <= 128) return f(std::integral_constant<int, 128>{});
  return f(std::integral_constant<int, 256>{});
}

template <typename F>
auto by_type(int dtype, F&& f) {
  return dtype == FR_F32 ? f(float{}) : f(bf16_t{});
}

template <typename T>
Rows<T> rows_of(const T* src, int64_t ld, int64_t n, int64_t n_out, int d, int D, bf16_t* out, float* inv) {
  Rows<T> r{};
  r.src = src;
  r.ld = ld;
  r.n = n;
  r.n_out = n_out;
  r.vec = d == D && ld % fr::kVec<T> == 0 && fr::aligned16(src);
  r.out = out;
  r.inv = inv;
  return r;
}

template <typename T, int D, bool GRAD>
void make_rows(const Rows<T>& h, const Rows<T>& w, int d, hipStream_t s) {
  const int64_t groups = (h.src ? fr::ceil_div(h.n_out, 32) : 0) + (w.src ? fr::ceil_div(w.n_out, 32) : 0);
  if (groups)
    hipLaunchKernelGGL((rows_kernel<T, D, GRAD>), fr::many_blocks(fr::ceil_div(groups, D >= 64 ? 1 : 2)), dim3(256), 0, s,
                       h, w, d);
}

template <typename T, int D, bool O>
void logp_fwd(const T* H, int64_t ldh, int64_t n, const T* W, int64_t ldw, int64_t nv, int d, const int64_t* ids, float c,
              float* logp, float* lse2, float* o, float* rest, void* ws, hipStream_t s) {
  const FwdWS w = fwd_ws<T, D, O>(ws, n, nv, d, ldw);
  const bool h_direct = direct<T>(d, D, ldh) && fr::aligned16(H), w_direct = direct<T>(d, D, ldw);
  Rows<T> h = rows_of<T>(h_direct ? nullptr : H, ldh, n, n, d, D, w.h, w.inv_h);
  h.ids = ids;
  h.nv = nv;
  make_rows<T, D, O>(h, rows_of<T>(w_direct ? nullptr : W, ldw, nv, nv, d, D, w.w, w.inv_w), d, s);
  StatsArgs a{};
  a.H = h_direct ? reinterpret_cast<const bf16_t*>(H) : w.h;
  a.ldh = h_direct ? ldh : D;
  a.part_h = n * D;
  a.n = n;
  a.W = w_direct ? reinterpret_cast<const bf16_t*>(W) : w.w;
  a.ldw = w_direct ? ldw : D;
  a.part_w = nv * D;
  a.nv = nv;
  a.inv_h = w.inv_h;
  a.inv_w = w.inv_w;
  if constexpr (sizeof(T) == 4) {
    a.rows_h = H;
    a.rows_w = W;
    a.ld_rows_h = ldh;
    a.ld_rows_w = ldw;
    a.d = d;
  }
  a.ids = ids;
  a.k = c * kLog2e;
  a.rt_n = w.sp.rt;
  a.sp_n = w.sp.sp;
  a.tiles_per_split = w.sp.per;
  a.stats = w.stats;
  a.o = w.o;
  const dim3 grid = fr::many_blocks(w.sp.blocks());
  if (w.nx == 2) {
    if constexpr (stats_blocks<T, D, O>() == 2) hipLaunchKernelGGL((stats_kernel<T, D, 2, O>), grid, dim3(256), 0, s, a);
  } else {
    hipLaunchKernelGGL((stats_kernel<T, D, 1, O>), grid, dim3(256), 0, s, a);
  }
  const FinishArgs f{w.stats, w.o, w.sp.sp, n, nv, ids, d, logp, lse2, o, rest};
  if (w.sp.sp >= kWideSplits && n <= kWideRows)
    hipLaunchKernelGGL((finish_kernel<D, O, true>), dim3((unsigned)n), dim3(1024), 0, s, f);
  else
    hipLaunchKernelGGL((finish_kernel<D, O, false>), fr::many_blocks(fr::ceil_div(n, 1024 / D)), dim3(256), 0, s, f);
}

template <typename T, int D>
void logp_dw(const T* H, int64_t ldh, int64_t n, const T* W, int64_t ldw, int64_t nv, int d, const int64_t* ids,
             const float* lse2, const float* rest, const float* up, float c, T* dW, void* ws, hipStream_t s) {
  const BwdWS w = bwd_ws<T, D>(ws, n, nv, d, ldw);
  const bool w_direct = direct<T>(d, D, ldw);
  Rows<T> h = rows_of<T>(H, ldh, n, w.n_pad, d, D, w.hs, w.inv_h);
  h.ids = ids;
  h.nv = nv;
  h.lse2 = lse2;
  h.rest = rest;
  h.up = up;
  h.c = c;
  h.lse_o = w.lse;
  h.coef = w.coef;
  h.target = w.target;
  h.ids_o = w.ids;
  make_rows<T, D, true>(h, rows_of<T>(w_direct ? nullptr : W, ldw, nv, nv, d, D, w.w, w.inv_w), d, s);
  GradArgs a{};
  a.X = w_direct ? reinterpret_cast<const bf16_t*>(W) : w.w;
  a.ldx = w_direct ? ldw : D;
  a.part_x = nv * D;
  a.nx = nv;
  a.inv_x = w.inv_w;
  a.Y = w.hs;
  a.ldy = D;
  a.part_y = w.n_pad * D;
  a.ny = w.n_pad;
  a.inv_y = w.inv_h;
  if constexpr (sizeof(T) == 4) {
    a.rows_x = W;
    a.rows_y = H;
    a.ld_rows_x = ldw;
    a.ld_rows_y = ldh;
    a.n = n;
  }
  a.lse = w.lse;
  a.coef = w.coef;
  a.target = w.target;
  a.ids = w.ids;
  a.lse2 = lse2;
  a.lse2_sum = lse2 + n;
  a.k = c * kLog2e;
  a.rt_n = w.v.rt;
  a.sp_n = w.v.sp;
  a.tiles_per_split = w.v.per;
  a.part = w.v.sp > 1 ? w.part : nullptr;
  a.out = dW;
  a.ldo = d;
  a.d = d;
  hipLaunchKernelGGL((grad_kernel<T, D>), fr::many_blocks(w.v.blocks()), dim3(256), 0, s, a);
  if (w.v.sp > 1)
    hipLaunchKernelGGL((join_kernel<T, D>), fr::many_blocks(fr::ceil_div(nv * (D / 4), 256)), dim3(256), 0, s, w.part,
                       w.v.sp, nv, dW, d);
}

}  // namespace

extern "C" int64_t fr_item_logp_fwd_workspace(int64_t n, int64_t n_items, int d, int64_t ldw, int dtype, int with_o) {
  if (!shape_ok(n, n_items, d)) return -1;
  return by_type(dtype, [&](auto t) {
    return by_width(d, [&](auto w) {
      using T = decltype(t);
      constexpr int D = decltype(w)::value;
      return with_o ? fwd_ws<T, D, true>(nullptr, n, n_items, d, ldw).bytes
                    : fwd_ws<T, D, false>(nullptr, n, n_items, d, ldw).bytes;
    });
  });
}

extern "C" int64_t fr_item_logp_bwd_workspace(int64_t n, int64_t n_items, int d, int64_t ldw, int dtype) {
  if (!shape_ok(n, n_items, d)) return -1;
  return by_type(dtype, [&](auto t) {
    return by_width(d, [&](auto w) { return bwd_ws<decltype(t), decltype(w)::value>(nullptr, n, n_items, d, ldw).bytes; });
  });
}

extern "C" int fr_item_logp_fwd(const void* d_h, int64_t ldh, int64_t n, const void* d_w, int64_t ldw, int64_t n_items,
                                int d, int dtype, const int64_t* d_ids, float scale, float* d_logp, float* d_lse2,
                                float* d_o, float* d_rest, void* d_workspace, int64_t workspace_bytes, void* stream) {
  FR_REQUIRE(dtype == FR_F32 || dtype == FR_BF16, "dtype must be FR_F32 or FR_BF16");
  FR_REQUIRE(shape_ok(n, n_items, d) && ldh >= d && ldw >= d, "bad shape (d in [1, 256])");
  FR_REQUIRE(scale > 0.f && scale < 1e30f, "scale must be positive");
  FR_REQUIRE(!d_o || d_rest, "d_o comes with d_rest");
  if (n == 0) return FR_OK;
  FR_REQUIRE(d_h && d_w && d_ids && d_logp && fr::aligned16(d_w), "null pointer, or the table not 16-byte aligned");
  FR_REQUIRE(d_workspace && fr::aligned16(d_workspace) &&
                 workspace_bytes >= fr_item_logp_fwd_workspace(n, n_items, d, ldw, dtype, d_o != nullptr),
             "workspace too small");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    by_width(d, [&](auto w) {
      constexpr int D = decltype(w)::value;
      const T *H = static_cast<const T*>(d_h), *W = static_cast<const T*>(d_w);
      if (d_o) logp_fwd<T, D, true>(H, ldh, n, W, ldw, n_items, d, d_ids, scale, d_logp, d_lse2, d_o, d_rest, d_workspace, s);
      else logp_fwd<T, D, false>(H, ldh, n, W, ldw, n_items, d, d_ids, scale, d_logp, d_lse2, d_o, d_rest, d_workspace, s);
    });
  });
  FR_LAUNCH_CHECK();
  return FR_OK;
}

extern "C" int fr_item_logp_bwd(const void* d_h, int64_t ldh, int64_t n, const void* d_w, int64_t ldw, int64_t n_items,
                                int d, int dtype, const int64_t* d_ids, const float* d_lse2, const float* d_o,
                                const float* d_rest, const float* d_up, float scale, void* d_dh, void* d_dw,
                                void* d_workspace, int64_t workspace_bytes, void* stream) {
  FR_REQUIRE(dtype == FR_F32 || dtype == FR_BF16, "dtype must be FR_F32 or FR_BF16");
  FR_REQUIRE(shape_ok(n, n_items, d) && n >= 1 && ldh >= d && ldw >= d, "bad shape (d in [1, 256])");
  FR_REQUIRE(scale > 0.f && scale < 1e30f, "scale must be positive");
  FR_REQUIRE(d_h && d_w && d_ids && d_up && (d_dh || d_dw) && fr::aligned16(d_w),
             "null pointer, or the table not 16-byte aligned");
  FR_REQUIRE(!d_dh || (d_o && d_rest), "dH needs the forward's d_o and d_rest");
  FR_REQUIRE(!d_dw || (d_lse2 && d_rest && d_workspace && fr::aligned16(d_workspace) &&
                       workspace_bytes >= fr_item_logp_bwd_workspace(n, n_items, d, ldw, dtype)),
             "dW needs the forward's d_lse2 and d_rest and a workspace");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    const T *H = static_cast<const T*>(d_h), *W = static_cast<const T*>(d_w);
    if (d_dh)
      hipLaunchKernelGGL(dh_kernel<T>, fr::many_blocks(fr::ceil_div(n * d, 256)), dim3(256), 0, s, d_o, d_rest, d_up, scale,
                         W, ldw, n_items, d_ids, n, d, static_cast<T*>(d_dh));
    if (d_dw)
      by_width(d, [&](auto w) {
        logp_dw<T, decltype(w)::value>(H, ldh, n, W, ldw, n_items, d, d_ids, d_lse2, d_rest, d_up, scale, static_cast<T*>(d_dw),
                                       d_workspace, s);
      });
  });
  FR_LAUNCH_CHECK();
  return FR_OK;
}

extern "C" int fr_preference_loss(const float* d_logp, const float* d_ref, const int64_t* d_offsets, int64_t pairs,
                                  int64_t n, float beta, float smoothing, float* d_loss, float* d_pair_loss,
                                  float* d_grad, void* stream) {
  FR_REQUIRE(pairs >= 1 && pairs < ((int64_t)1 << 31) && n >= 0, "bad shape");
  FR_REQUIRE(beta > 0.f && beta < INFINITY && smoothing >= 0.f && smoothing <= 0.5f,
             "beta must be positive and the label smoothing in [0, 1/2]");
  FR_REQUIRE(d_offsets && d_loss && d_pair_loss && (n == 0 || (d_logp && d_grad)), "null pointer");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (pairs <= kFewPairs && n <= kFewPositions) {
    hipLaunchKernelGGL(pairs_few_kernel, dim3(1), dim3(1024), 0, s, d_logp, d_ref, d_offsets, pairs, n, beta, smoothing,
                       d_loss, d_grad);
  } else {
    if (n)
      hipLaunchKernelGGL(clear_kernel, dim3((unsigned)std::min<int64_t>(fr::ceil_div(n, 256), 1024)), dim3(256), 0, s,
                         d_grad, n);
    hipLaunchKernelGGL(pair_kernel, fr::many_blocks(fr::ceil_div(pairs, 4)), dim3(256), 0, s, d_logp, d_ref, d_offsets,
                       pairs, n, beta, smoothing, d_pair_loss, d_grad);
    hipLaunchKernelGGL(pair_mean_kernel, dim3(1), dim3(1024), 0, s, d_pair_loss, pairs, d_loss);
  }
  FR_LAUNCH_CHECK();
  return FR_OK;
}
