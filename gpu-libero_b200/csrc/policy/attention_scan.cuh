// The trajectory form of decay attention on tensor cores.
//
// Tokens are taken in chunks of 64.  With S the state before a chunk of n
// tokens and lambda the head's decay,
//   out_i = sum_{j <= i} lambda^(i-j) (q_i . k_j) v_j + lambda^(i+1) q_i S
//   S'    = lambda^n S + sum_j lambda^(n-1-j) k_j v_j^T
// so a chunk is four products: Q K^T, (weighted) P V, Q S and (weighted K)^T V.
// A scan that runs backward is the same with its tokens in reverse order; there
// the state decays after a token instead of before it: lambda^i for Q S and
// lambda^(n-j) for S'.  An episode's start cuts the sums: weights between
// tokens of different episodes are zero.  So that nothing of a diverged world
// reaches its next episode (or the tokens before it diverged) through a product
// of zero and infinity, rows and states that are not finite are summed again
// over their own tokens alone.
//
// Four warps own 16 query rows each, and 1/4 of S in registers as the
// accumulator of K^T V; S passes through shared memory for Q S.  P stays in
// registers: the accumulator layout of one product is the operand layout of the
// next.  A CTA owns one row, head, 64-wide slice of v and (for few long rows)
// one piece of the row, and walks the chunks; the next chunk's loads fly meanwhile.
//
// What bounds it: not one unit alone.  For 1184 rows of 256 tokens and 4 heads of 64
// in bf16 (215 us forward, 56% of the copy bandwidth; 750 us with the gradients) the
// tensor pipe is busy 39% of the time, the instruction slots half of it and shared
// memory's pipe 60%, with 16 warps an SM; what is left are the warps' waits for each
// other's and their own results.  The main loop has to fit the instruction cache:
// taking the rare paths out of line, and a variant for full tiles, took the training
// pass from 931 us to 789.
//
// Roundings, beside the output's: bf16 rounds P and the copy of S that a chunk
// reads to bf16 (one rounding each of the output's own size).  The weighted K
// is split into PARTS bf16 terms: three are exact to 2^-24, as a state that
// leaves in 32 bits needs (two would leave the square of bf16's mean rounding,
// 2.6e-6); two where the state only feeds 16-bit outputs.  fp16 does those three
// products in tf32 (P and S rounded to its 11 bits, weighted K in two terms), which
// has fp16's precision without its range: a sum of products overflows fp16 easily.
// fp32 splits every operand into two tf32 terms and keeps three of the four products.
#pragma once
#include "attention_scan.h"
#include "common.cuh"
#include <type_traits>

namespace b200policy {
namespace scan {

// ---- matrix products: 16 x 8 += 16 x 16 . 16 x 8 -----------------------------
// Lane = 4 g + t.  Accumulator: rows g, g + 8, columns 2t, 2t + 1.  A values in
// the order (g, 2t) (g, 2t+1) (g+8, 2t) (g+8, 2t+1) and the same with 8 added
// to the second index; B values (2t, g) (2t+1, g) (2t+8, g) (2t+9, g).  A tf32
// product takes them as two steps of depth 8 whose inner index is permuted.
__device__ __forceinline__ void mma(float c[4], const uint32_t a[4], const uint32_t b[2], __nv_bfloat16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma(float c[4], const uint32_t a[4], const uint32_t b[2], __half) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// a, b: eight and four values of the order above; both depth-8 steps.
__device__ __forceinline__ void mma_tf32(float c[4], const uint32_t a[8], const uint32_t b[4]) {
#pragma unroll
  for (int s = 0; s < 2; ++s)
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[4 * s]), "r"(a[4 * s + 2]), "r"(a[4 * s + 1]), "r"(a[4 * s + 3]), "r"(b[2 * s]), "r"(b[2 * s + 1]));
}

__device__ __forceinline__ uint32_t tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ uint32_t pack(float lo, float hi, __half) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ float2 unpack(uint32_t r, __nv_bfloat16) {
  return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack(uint32_t r, __half) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&r));
}

// Fragments of tensors' own values.
template <class T> struct A16 {
  uint32_t r[4];
  __device__ __forceinline__ void values(F2 x[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack(r[i], T());
      x[i] = F2(f.x, f.y);
    }
  }
};
template <> struct A16<float> {
  float r[8];
  __device__ __forceinline__ void values(F2 x[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = F2(r[2 * i], r[2 * i + 1]);
  }
};
template <class T> struct B16 {
  uint32_t r[2];
  __device__ __forceinline__ void values(float x[4]) const {
    const float2 a = unpack(r[0], T()), b = unpack(r[1], T());
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
  }
};
template <> struct B16<float> {
  float r[4];
  __device__ __forceinline__ void values(float x[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = r[i];
  }
};

__device__ __forceinline__ void flat(float x[8], const F2 v[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = v[i].get().x, x[2 * i + 1] = v[i].get().y;
}

// Two tf32 terms of N values.
template <int N> struct Pair {
  uint32_t hi[N], lo[N];
  __device__ __forceinline__ explicit Pair(const F2 *v) {
    float x[N];
    flat(x, v);
    *this = Pair(x);
  }
  __device__ __forceinline__ explicit Pair(const float x[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      hi[i] = tf32(x[i]);
      lo[i] = __float_as_uint(x[i] - __uint_as_float(hi[i]));
    }
  }
};
__device__ __forceinline__ void mma_pairs(float c[4], const Pair<8> &a, const Pair<4> &b) {
  mma_tf32(c, a.lo, b.hi);
  mma_tf32(c, a.hi, b.lo);
  mma_tf32(c, a.hi, b.hi);
}

// Computed values (P, weighted K) as an A operand against a tensor's values, in
// `parts` <= PARTS terms.  mul() runs over N accumulators term by term, so that
// consecutive products do not wait for each other.
template <class T, int PARTS> struct Value;
template <int PARTS> struct Value<__nv_bfloat16, PARTS> {
  uint32_t r[PARTS][4];
  __device__ __forceinline__ explicit Value(F2 x[4], int parts = PARTS) {
    const F2 less(-1.f);
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
      if (p < 2 || p < parts)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          r[p][i] = pack(x[i].get().x, x[i].get().y, __nv_bfloat16());
          if (p + 1 < PARTS) {
            const float2 f = unpack(r[p][i], __nv_bfloat16());
            x[i] = fma(F2(f.x, f.y), less, x[i]);
          }
        }
  }
  template <int N> __device__ __forceinline__ void mul(float (*c)[4], const B16<__nv_bfloat16> *b, int parts) const {
#pragma unroll
    for (int p = PARTS - 1; p >= 0; --p)
      if (p < 2 || p < parts)
#pragma unroll
        for (int j = 0; j < N; ++j) mma(c[j], r[p], b[j].r, __nv_bfloat16());
  }
};
template <int PARTS> struct Value<__half, PARTS> {
  uint32_t r[PARTS][8];
  __device__ __forceinline__ explicit Value(const F2 v[4], int = PARTS) {
    float x[8];
    flat(x, v);
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        r[p][i] = tf32(x[i]);
        x[i] -= __uint_as_float(r[p][i]);
      }
  }
  template <int N> __device__ __forceinline__ void mul(float (*c)[4], const B16<__half> *b, int) const {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float y[4];
      b[j].values(y);
      const uint32_t v[4] = {__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])};
#pragma unroll
      for (int p = PARTS - 1; p >= 0; --p) mma_tf32(c[j], r[p], v);
    }
  }
};
template <int PARTS> struct Value<float, PARTS> {
  Pair<8> a;
  __device__ __forceinline__ explicit Value(const F2 v[4], int = PARTS) : a(v) {}
  template <int N> __device__ __forceinline__ void mul(float (*c)[4], const B16<float> *b, int) const {
#pragma unroll
    for (int j = 0; j < N; ++j) mma_pairs(c[j], a, Pair<4>(b[j].r));
  }
};

// Tensor values against tensor values.
template <class T> __device__ __forceinline__ void mma_exact(float c[4], const A16<T> &a, const B16<T> &b) {
  mma(c, a.r, b.r, T());
}
__device__ __forceinline__ void mma_exact(float c[4], const A16<float> &a, const B16<float> &b) {
  mma_pairs(c, Pair<8>(a.r), Pair<4>(b.r));
}

// ---- shared memory -----------------------------------------------------------
__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <bool TRANS> __device__ __forceinline__ void ldmatrix(uint32_t r[4], uint32_t at) {
  if (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at));
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at));
}

// A tile of W columns.  16-bit: 16-byte blocks permuted by their row, so that
// eight rows of one column block lie in different banks; the permutation is an
// exclusive or of address bits, so a lane's address for any 16 x 16 part is one
// of two lane addresses, xored with the part's columns, plus its rows.  32-bit:
// PAD more columns: 8 for tiles read along their rows, 4 along columns.
template <class T, int W, int PAD> struct Tile {
  static constexpr int kPitch = sizeof(T) == 2 ? W : W + PAD;
  static constexpr int kBlock = 16 / sizeof(T);  // elements of 16 bytes
  static constexpr bool kTurns = sizeof(T) == 2 && W >= 64;
  T *p;
  uint32_t a, b;  // 16-bit: shared addresses of the lane's rows for the two kinds of part
  static __device__ __forceinline__ int at(int row, int col) {
    if (sizeof(T) == 4) return row * kPitch + col;
    const int turn = W >= 64 ? row & 7 : (row >> 1) & 3;
    return row * W + ((((col >> 3) ^ turn) << 3) | (col & 7));
  }
  static constexpr int bytes(int rows) { return rows * kPitch * (int)sizeof(T); }
  __device__ __forceinline__ Tile(T *p, int lane) : p(p), a(0), b(0) {
    if (sizeof(T) == 2) {
      a = smem_addr(p + at(lane & 15, (lane >> 4) * 8));
      b = smem_addr(p + at((lane & 7) + (lane >> 4) * 8, ((lane >> 3) & 1) * 8));
    }
  }

  // a 16-bit tile of the same width
  template <int PAD2> __device__ __forceinline__ explicit Tile(const Tile<T, W, PAD2> &o) : p(o.p), a(o.a), b(o.b) {}

  __device__ __forceinline__ Tile behind(int bytes) const {
    Tile r = *this;
    r.p = (T *)((unsigned char *)p + bytes), r.a += bytes, r.b += bytes;
    return r;
  }

  // rows r0 .. r0+15 as A, inner index k0 .. k0+15
  __device__ __forceinline__ A16<T> rows_a(int r0, int k0, int lane) const {
    A16<T> x;
    if constexpr (sizeof(T) == 2) {
      ldmatrix<false>(x.r, (a ^ (k0 * 2)) + r0 * W * 2);
    } else {
      const int g = lane >> 2, t = lane & 3;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 u = *(const float2 *)(p + at(r0 + g, k0 + 2 * t + 8 * h));
        const float2 v = *(const float2 *)(p + at(r0 + g + 8, k0 + 2 * t + 8 * h));
        x.r[4 * h] = u.x, x.r[4 * h + 1] = u.y, x.r[4 * h + 2] = v.x, x.r[4 * h + 3] = v.y;
      }
    }
    return x;
  }
  // columns m0 .. m0+15 as A's rows, inner index = rows r0 .. r0+15
  __device__ __forceinline__ A16<T> columns_a(int r0, int m0, int lane) const {
    A16<T> x;
    if constexpr (sizeof(T) == 2) {
      ldmatrix<true>(x.r, (b ^ (m0 * 2)) + r0 * W * 2);
    } else {
      const int g = lane >> 2, t = lane & 3;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x.r[4 * h + e] = p[at(r0 + 2 * t + 8 * h + (e & 1), m0 + g + 8 * (e >> 1))];
    }
    return x;
  }
  // rows n0 .. n0+15 as the columns of two B operands, inner index k0 .. k0+15
  __device__ __forceinline__ void rows_b(B16<T> y[2], int n0, int k0, int lane) const {
    if constexpr (sizeof(T) == 2) {
      uint32_t r[4];
      ldmatrix<false>(r, (b ^ (k0 * 2)) + n0 * W * 2);
      y[0].r[0] = r[0], y[0].r[1] = r[1], y[1].r[0] = r[2], y[1].r[1] = r[3];
    } else {
      const int g = lane >> 2, t = lane & 3;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 x = *(const float2 *)(p + at(n0 + 8 * i + g, k0 + 2 * t + 8 * h));
          y[i].r[2 * h] = x.x, y[i].r[2 * h + 1] = x.y;
        }
    }
  }
  // columns n0 .. n0+15 as two B operands, inner index = rows k0 .. k0+15
  __device__ __forceinline__ void columns_b(B16<T> y[2], int k0, int n0, int lane) const {
    if constexpr (sizeof(T) == 2) {
      uint32_t r[4];
      ldmatrix<true>(r, (a ^ (n0 * 2)) + k0 * W * 2);
      y[0].r[0] = r[0], y[0].r[1] = r[1], y[1].r[0] = r[2], y[1].r[1] = r[3];
    } else {
      const int g = lane >> 2, t = lane & 3;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[i].r[e] = p[at(k0 + 2 * t + 8 * (e >> 1) + (e & 1), n0 + 8 * i + g)];
    }
  }
  // the pair of accumulator columns 8j + 2t of rows r0 + g and r0 + g + 8
  __device__ __forceinline__ void put(int r0, int j, int lane, float x0, float x1, float y0, float y1) const {
    const int g = lane >> 2, t = lane & 3;
    if constexpr (sizeof(T) == 2) {
      const uint32_t to = (smem_addr(p + at(g, 2 * t)) ^ (j * 16)) + r0 * W * 2;
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(to), "r"(pack(x0, x1, T())) : "memory");
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + 8 * W * 2), "r"(pack(y0, y1, T())) : "memory");
    } else {
      *(float2 *)(p + at(r0 + g, 8 * j + 2 * t)) = make_float2(x0, x1);
      *(float2 *)(p + at(r0 + g + 8, 8 * j + 2 * t)) = make_float2(y0, y1);
    }
  }
};

__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(take ? 16 : 0));
}
__device__ __forceinline__ void scale(float c[4], F2 x, F2 y) {
  const float2 u = mul(F2(c[0], c[1]), x).get(), v = mul(F2(c[2], c[3]), y).get();
  c[0] = u.x, c[1] = u.y, c[2] = v.x, c[3] = v.y;
}
// Whether every value of a lane's accumulators is finite, in the whole warp.
template <int N> __device__ __forceinline__ bool all_finite(const float (*c)[4]) {
  F2 x;
#pragma unroll
  for (int j = 0; j < N; ++j) x = fma(F2(c[j][0], c[j][1]), F2(), fma(F2(c[j][2], c[j][3]), F2(), x));
  return __all_sync(~0u, x.sum() == 0.f);
}
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// The copy where 16-byte accesses are not aligned; out of line, since the main
// loop's code has to stay small for the instruction cache.  A warp takes its own 16
// rows, 32 columns at a time.  Values of 4 bytes are copied past the registers, all
// of them at once; of 2 bytes, sixteen are on their way.
template <class T, class TILE, int COLS>
__device__ __noinline__ void load_single(T *tile, const T *from, int64_t stride, int rows, int width) {
  const int lane = threadIdx.x & 31, top = threadIdx.x / 32 * 16;
  constexpr int kAcross = COLS / 32, kAtOnce = 16 / kAcross;
  from += top * stride + lane;
#pragma unroll 1
  for (int r0 = top; r0 < top + 16; r0 += kAtOnce) {
    T x[kAtOnce][kAcross];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i, from += stride)
#pragma unroll
      for (int j = 0; j < kAcross; ++j) {
        const int r = r0 + i, c = lane + 32 * j;
        const bool take = r < rows && c < width;
        if constexpr (sizeof(T) == 4)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_addr(tile + TILE::at(r, c))),
                       "l"(take ? from + 32 * j : from - r * stride - lane), "r"(take ? 4 : 0)
                       : "memory");
        else
          x[i][j] = take ? from[32 * j] : from_float<T>(0.f);
      }
    if constexpr (sizeof(T) == 2)
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
        for (int j = 0; j < kAcross; ++j) tile[TILE::at(r0 + i, lane + 32 * j)] = x[i][j];
  }
}

// One tensor's way into its tile: rows of `stride` from `base` (advanced chunk by
// chunk), the first `rows` of them and the first `width` columns; the rest of the
// tile's COLS columns is zero.  Every warp fetches its own 16 rows.
template <class T, class TILE, int COLS, int MODE> struct Loader {
  static constexpr bool FULL = MODE == 2, VEC = MODE >= 1;
  static constexpr int kBlocks = COLS / TILE::kBlock, kRows = 32 / kBlocks, kSteps = 16 / kRows;
  const T *base;  // of this thread's first block where copies are 16 bytes, else of the tile
  int64_t stride;
  bool vec, in;
  int width;
  __device__ __forceinline__ Loader(const T *from, int64_t stride, int width, bool vec)
      : base(from), stride(stride), vec(vec), width(width) {
    const int col = threadIdx.x % kBlocks * TILE::kBlock;
    in = FULL || col < width;
    if (VEC || vec) base += row() * stride + (in ? col : 0);
  }
  static __device__ __forceinline__ int row() { return threadIdx.x / 32 * 16 + threadIdx.x % 32 / kBlocks; }
  __device__ __forceinline__ void load(const TILE &tile, int chunk, int rows) const {
    const T *from = base + (int64_t)chunk * kTile * stride;
    if (VEC || vec) {
      const uint32_t to = smem_addr(tile.p + TILE::at(row(), threadIdx.x % kBlocks * TILE::kBlock));
      // rows of a permuted tile: the row's turn changes the block's address bits
      auto at = [&](int i) {
        return (to ^ (TILE::kTurns ? (i * kRows & 7) * 16 : 0)) + i * kRows * TILE::kPitch * (int)sizeof(T);
      };
      if (in && rows == kTile) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i, from += kRows * stride) copy16(at(i), from, true);
      } else {
#pragma unroll
        for (int i = 0; i < kSteps; ++i, from += kRows * stride) {
          const bool take = in && row() + i * kRows < rows;
          copy16(at(i), take ? from : base, take);
        }
      }
    } else {
      load_single<T, TILE, COLS>(tile.p, from, stride, rows, width);
    }
  }
};

// ---- the kernel --------------------------------------------------------------
template <class T, int KT, int VT, bool TWIN> struct Layout {
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr bool kState16 = std::is_same<T, __nv_bfloat16>::value;  // S in shared memory
  using State = typename std::conditional<kState16, __nv_bfloat16, float>::type;
  // the query tile also stages the output rows
  using Q = Tile<T, (KT > VT ? KT : VT), 8>;
  using K = Tile<T, KT, 8>;
  using V = Tile<T, VT, 4>;
  using S = Tile<State, VT, 4>;
  static constexpr int kQ = Q::bytes(kTile), kK = K::bytes(kTile), kV = V::bytes(kTile), kS = S::bytes(KT);
  // Two buffers of K and V where four CTAs still fit with them; Q has one, as every
  // warp fetches its own next rows when it has done with the present ones.
  static constexpr int kStages = kState16 && KT <= 64 && !TWIN ? 2 : 1, kStage = kK + kV;
  // three tables of lambda^m for m of 0 to kTile, each behind 16 zeros (the first
  // needs none: a whole chunk's decay lies there)
  static constexpr int kTable = 16 + kTile + 1;
  static constexpr int kX = kQ, kTiles = kQ + (TWIN ? kQ : 0) + kStages * kStage;  // X: a twin's queries
  static constexpr int kBytes = kTiles + kS + 3 * kTable * 4 + 2 * 4;
  // CTAs of one SM, by shared memory (of 228 KB, 1 KB more for each CTA); more
  // than four would leave too few registers
  static constexpr int kFit = 228 * 1024 / (kBytes + 1024);
  static constexpr int kResident = kFit < 1 ? 1 : kFit > 4 ? 4 : kFit;
};

// A product with weight zero is zero only if its factors are finite.  These sum
// four of a lane's accumulators (rows r and r + 8, columns col and col + 1) over
// their own tokens alone; out of line, as they hardly ever run.
template <class T, class L>
__device__ __noinline__ float4 row_sums(const T *q, const T *k, const T *v, const typename L::State *S, int r, int col,
                                        int2 low, int carried, int kd, const float *into, const float *within, bool turned) {
  float sum[4];
#pragma unroll 1
  for (int e = 0; e < 4; ++e) {
    const int i = r + (e & 2 ? 8 : 0), c = col + (e & 1);
    float x = 0.f;
    if (carried & (e & 2 ? 2 : 1)) {
#pragma unroll 1
      for (int d = 0; d < kd; ++d) x += to_float(q[L::Q::at(i, d)]) * to_float(S[turned ? L::S::at(c, d) : L::S::at(d, c)]);
      x *= into[i];
    }
#pragma unroll 1
    for (int j = e & 2 ? low.y : low.x; j <= i; ++j) {
      float dot = 0.f;
#pragma unroll 1
      for (int d = 0; d < kd; ++d) dot += to_float(q[L::Q::at(i, d)]) * to_float(k[L::K::at(j, d)]);
      x += dot * within[i - j] * to_float(v[L::V::at(j, c)]);
    }
    sum[e] = x;
  }
  return make_float4(sum[0], sum[1], sum[2], sum[3]);
}
template <class T, class L>
__device__ __noinline__ float4 state_sums(const T *k, const T *v, int low, int rows, int r, int col, const float *kept) {
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int j = low; j < rows; ++j) {
    const float k0 = to_float(k[L::K::at(j, r)]) * kept[-j], k1 = to_float(k[L::K::at(j, r + 8)]) * kept[-j];
    const float v0 = to_float(v[L::V::at(j, col)]), v1 = to_float(v[L::V::at(j, col + 1)]);
    sum.x += k0 * v0, sum.y += k0 * v1, sum.z += k1 * v0, sum.w += k1 * v1;
  }
  return sum;
}

// Rows of a staged tile to their places where 16-byte accesses are not aligned.
template <class T, class TILE>
__device__ __noinline__ void store_single(const T *tile, T *to, int64_t stride, int rows, int width) {
#pragma unroll 1
  for (int i = 0; i < rows; ++i, to += stride)
    for (int col = threadIdx.x & 31; col < width; col += 32) to[col] = tile[TILE::at(i, col)];
}

// MODE: 0 any sizes and alignment; 1 16-byte accesses throughout; 2 also every tensor
// fills its tiles and leaves in its own type.
template <class T, int KT, int VT, int PARTS, int MODE, bool TWIN>
__global__ void __launch_bounds__(kScanThreads, Layout<T, KT, VT, TWIN>::kResident)
    scan_kernel(const __grid_constant__ ScanParams p) {
  constexpr bool FULL = MODE == 2, VEC = MODE >= 1;
  using L = Layout<T, KT, VT, TWIN>;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *states = smem + L::kTiles;
  float *into = (float *)(states + L::kS) + 16;  // lambda^m out_scale: the state's weight in a row
  float *within = into + L::kTable;                           // lambda^m pair_scale out_scale: a key's weight in a row
  float *kept = within + L::kTable;                           // lambda^m pair_scale: a key's weight in the state
  unsigned *marks = (unsigned *)(kept + kTile + 1);  // [half of the chunk]: tokens that start an episode
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const typename L::Q tile_q((T *)smem, lane);
  const typename L::K tile_k((T *)(smem + L::kTiles - L::kStages * L::kStage), lane);
  const typename L::V tile_v((T *)(smem + L::kTiles - L::kStages * L::kStage + L::kK), lane);
  const typename L::Q tile_x((T *)(smem + L::kX), lane);
  const typename L::S tile_s((typename L::State *)states, lane);

  // which scan, slice, piece, head and row
  int unit = blockIdx.x % p.units, which = 0;
  while (unit >= p.scan[which].slices) unit -= p.scan[which++].slices;
  const Scan &s = p.scan[which];
  const int v0 = unit * VT, kd = FULL ? KT : s.kd, vd = FULL ? VT : min(VT, s.vd - v0);
  const int rest = blockIdx.x / p.units, piece = rest % p.pieces, bh = rest / p.pieces;
  const int b = bh / p.heads, h = bh % p.heads, shared_h = h / p.group;
  const int n = p.lengths ? min(max(p.lengths[b], 0), p.time) : p.time;
  const int s0 = piece * p.piece, own = min(max(n - s0, 0), p.piece);
  const int chunks = (own + kTile - 1) / kTile;

  // the scan's token i is the row's token i, or n - 1 - i
  const int step = s.reverse ? -1 : 1, lag = s.reverse ? 0 : 1;
  const int origin = s.reverse ? n - 1 - s0 : s0;
  const Loader<T, typename L::Q, KT, MODE> load_q(
      (const T *)s.q + b * s.q_batch + (s.q_shared ? shared_h : h) * s.q_head + origin * s.q_time, step * s.q_time, kd,
      s.vec_q);
  const Loader<T, typename L::K, KT, MODE> load_k(
      (const T *)s.k + b * s.k_batch + (s.k_shared ? shared_h : h) * s.k_head + origin * s.k_time, step * s.k_time, kd,
      s.vec_k);
  const Loader<T, typename L::V, VT, MODE> load_v(
      (const T *)s.v + b * s.v_batch + (s.v_shared ? shared_h : h) * s.v_head + origin * s.v_time + v0,
      step * s.v_time, vd, s.vec_v);
  auto load_queries = [&](int c) {
    if (p.state_only) return;
    const int rows = min(kTile, own - c * kTile);
    load_q.load(tile_q, c, rows);
    if constexpr (TWIN)
      Loader<T, typename L::Q, KT, MODE>(
          (const T *)s.x + b * s.x_batch + (s.x_shared ? shared_h : h) * s.x_head + origin * s.x_time, step * s.x_time, s.vd,
          s.vec_x)
          .load(tile_x, c, rows);
  };
  auto load_keys = [&](int c) {
    const int rows = min(kTile, own - c * kTile), to = L::kStages == 2 ? (c & 1) * L::kStage : 0;
    load_k.load(tile_k.behind(to), c, rows);
    load_v.load(tile_v.behind(to), c, rows);
  };
  auto starts = [&](int c) {  // of token tid (< kTile) of chunk c
    const int i = c * kTile + tid;
    return p.first && tid < kTile && i < own && p.first[b * p.first_batch + (origin + step * i) * p.first_time];
  };
  auto mark = [&](bool start) {
    const unsigned m = __ballot_sync(~0u, start);
    if (lane == 0 && warp < kTile / 32) marks[warp] = m;
  };
  if (chunks) load_queries(0), load_keys(0);

  const float log_decay = p.log_decay[h];
  if (tid < L::kTable) {
    const int m = tid - 16;
    const float x = m > 0 ? expf(log_decay * m) : m == 0 ? 1.f : 0.f;
    if (m >= 0) into[m] = x * s.out_scale;
    within[m] = x * s.pair_scale * s.out_scale;
    kept[m] = x * s.pair_scale;
  }
  Decay *whole = (Decay *)(into - 16);
  if (tid == 0) *whole = Decay(log_decay * kTile);

  // S: warp owns kM tiles of 16 rows and kN tiles of 8 columns
  constexpr int kM = KT >= 64 ? KT / 64 : 1, kN = KT >= 64 ? VT / 8 : VT / 16;
  const int m0 = KT >= 64 ? warp * kM * 16 : (warp & 1) * 16, n0 = KT >= 64 ? 0 : (warp >> 1) * kN * 8;
  float S[kM][kN][4];
  {
    const float *init = s.init;
    int row = (int)s.init_row, col = (int)s.init_col;
    if (init) init += (int64_t)bh * kd * s.vd;
    if (p.state_only) init = nullptr;
    else if (p.pieces > 1) {
      init = p.states + p.states_at[which] + ((int64_t)bh * p.pieces + piece) * kd * s.vd;
      row = s.vd, col = 1;
    }
    const int top = m0 + g, left = n0 + 2 * t;
    if (!init) {
#pragma unroll
      for (int i = 0; i < kM; ++i)
#pragma unroll
        for (int j = 0; j < kN; ++j) S[i][j][0] = S[i][j][1] = S[i][j][2] = S[i][j][3] = 0.f;
    } else {
      init += top * row + (v0 + left) * col;
      const bool whole = kd == KT && vd == VT;
#pragma unroll
      for (int j = 0; j < kN; ++j, init += 8 * col) {
        const float *at = init;
#pragma unroll
        for (int i = 0; i < kM; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half, at += 8 * row) {
            const bool in = whole || top + 16 * i + 8 * half < kd;
            S[i][j][2 * half] = in && (whole || left + 8 * j < vd) ? at[0] : 0.f;
            S[i][j][2 * half + 1] = in && (whole || left + 8 * j + 1 < vd) ? at[col] : 0.f;
          }
      }
    }
  }
  auto publish = [&] {
#pragma unroll
    for (int i = 0; i < kM; ++i)
#pragma unroll
      for (int j = 0; j < kN; ++j)
        tile_s.put(m0 + 16 * i, n0 / 8 + j, lane, S[i][j][0], S[i][j][1], S[i][j][2], S[i][j][3]);
  };
  if (chunks) mark(starts(0));
  if (!p.state_only) publish();

  bool cut = false;  // an episode started in this piece
#pragma unroll 1
  for (int c = 0; c < chunks; ++c) {
    copy_wait();
    __syncthreads();
    bool next = false;
    if (c + 1 < chunks) {
      next = starts(c + 1);
      if (L::kStages == 2) load_keys(c + 1);
    }
    const int rows = min(kTile, own - c * kTile);
    const unsigned long long flags = marks[0] | (unsigned long long)marks[1] << 32;
    // The first token that token i's sums reach: where its episode starts.  A
    // start counts for its own token in token order, and for those behind it in
    // the reverse order.  Zero where the episode is older than the chunk.
    auto reach = [&](int i) {
      const unsigned long long before = flags & ((lag ? 2ull << i : 1ull << i) - 1);
      return before ? 64 - lag - __clzll(before) : 0;
    };
    auto carried = [&](int i) { return !(flags & ((lag ? 2ull << i : 1ull << i) - 1)); };
    const int last = flags ? 64 - lag - __clzll(flags) : 0;  // the first token that the state after the chunk holds
    const auto K = tile_k.behind(L::kStages == 2 ? (c & 1) * L::kStage : 0);
    const auto V = tile_v.behind(L::kStages == 2 ? (c & 1) * L::kStage : 0);
    const int r0 = 16 * warp + g, r1 = r0 + 8;  // this lane's query rows
    if (!p.state_only && 16 * warp < rows) {
      const int reach0 = flags ? reach(r0) : 0, reach1 = flags ? reach(r1) : 0;
      // the output, and its twin with S turned and K and V in each other's place
#pragma unroll 1
      for (int pass = 0; pass < (TWIN ? 2 : 1); ++pass) {
        const bool turned = TWIN && pass;
        const typename L::Q Q = turned ? tile_x : tile_q;
        typename L::K Ks = K;
        typename L::V Vs = V;
        if constexpr (TWIN)
          if (turned) Ks = typename L::K(V), Vs = typename L::V(K);
        const int depth = FULL ? KT : turned ? s.vd : kd, width = FULL ? VT : turned ? kd : vd, across = turned ? kd : s.vd;
        void *out_to = turned ? s.twin_out : s.out;
        const bool vec_out = turned ? s.vec_twin : s.vec_out;
        float o[VT / 8][4];
#pragma unroll
        for (int j = 0; j < VT / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        // Q S
#pragma unroll(L::kWide ? 1 : KT / 16)
        for (int ks = 0; ks < KT / 16; ++ks) {
          if (!FULL && 16 * ks >= depth) break;
          const A16<T> a = Q.rows_a(16 * warp, 16 * ks, lane);
#pragma unroll
          for (int j = 0; j < VT / 8; j += 2) {
            B16<typename L::State> sb[2];
            if (turned) tile_s.rows_b(sb, 8 * j, 16 * ks, lane);
            else tile_s.columns_b(sb, 16 * ks, 8 * j, lane);
            if constexpr (std::is_same<T, __half>::value) {
              float x[8];
              uint32_t xa[8];
              F2 xv[4];
              a.values(xv);
              flat(x, xv);
#pragma unroll
              for (int e = 0; e < 8; ++e) xa[e] = __float_as_uint(x[e]);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                uint32_t y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = tf32(sb[i].r[e]);
                mma_tf32(o[j + i], xa, y);
              }
            } else {
              mma_exact(o[j], a, sb[0]);
              mma_exact(o[j + 1], a, sb[1]);
            }
          }
        }
        {
          const float w0 = flags && !carried(r0) ? 0.f : into[r0 + lag];
          const float w1 = flags && !carried(r1) ? 0.f : into[r1 + lag];
#pragma unroll
          for (int j = 0; j < VT / 8; ++j) scale(o[j], F2(w0), F2(w1));
        }
        // P = weighted Q K^T, 16 keys at a time, then P V
        const float *w = within + r0 - 2 * t;
        int key = 2 * t;
#pragma unroll 1
        for (int kt = 0; kt <= warp; ++kt, w -= 16, key += 16) {
          float pr[2][4] = {};
#pragma unroll(L::kWide ? 1 : KT / 16)
          for (int ks = 0; ks < KT / 16; ++ks) {
            if (!FULL && 16 * ks >= depth) break;
            const A16<T> a = Q.rows_a(16 * warp, 16 * ks, lane);
            B16<T> kb[2];
            Ks.rows_b(kb, 16 * kt, 16 * ks, lane);
            mma_exact(pr[0], a, kb[0]);
            mma_exact(pr[1], a, kb[1]);
          }
          F2 x[4];  // rows r0, r1 of keys 2t, 2t + 1, and of 2t + 8, 2t + 9
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float *wi = w + (i & 1 ? 8 : 0) - 8 * (i >> 1);
            x[i] = mul(F2(pr[i >> 1][2 * (i & 1)], pr[i >> 1][2 * (i & 1) + 1]), F2(wi[0], wi[-1]));
          }
          if (flags)  // (the table holds zeros for tokens behind the row's own)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int j = key + 8 * (i >> 1), low = i & 1 ? reach1 : reach0;
              x[i] = F2(j >= low ? x[i].get().x : 0.f, j + 1 >= low ? x[i].get().y : 0.f);
            }
          const Value<T, 1> pv(x);
          B16<T> vb[VT / 8];
#pragma unroll
          for (int j = 0; j < VT / 8; j += 2) Vs.columns_b(vb + j, 16 * kt, 8 * j, lane);
          pv.template mul<VT / 8>(o, vb, 1);
        }
        if (!all_finite<VT / 8>(o)) {
#pragma unroll
          for (int j = 0; j < VT / 8; ++j)
            *(float4 *)o[j] = row_sums<T, L>(Q.p, Ks.p, Vs.p, tile_s.p, r0, 8 * j + 2 * t, make_int2(reach0, reach1),
                                             flags ? carried(r0) + 2 * carried(r1) : 3, depth, into + lag, within, turned);
          __syncwarp();
        }
        // out: this warp's rows from `first`, `stride` apart
        const int64_t stride = (int64_t)step * p.heads * across;
        const int64_t first = (((int64_t)b * p.time + origin + step * (c * kTile + 16 * warp)) * p.heads + h) * across + v0;
        const int count = min(16, rows - 16 * warp);
        if (sizeof(T) == 4 || (!FULL && s.out_float)) {
          float *to = (float *)out_to + first + g * stride + 2 * t;
#pragma unroll
          for (int half = 0; half < 2; ++half, to += 8 * stride) {
            if (g + 8 * half >= count) continue;
#pragma unroll
            for (int j = 0; j < VT / 8; ++j) {
              const int room = width - 8 * j - 2 * t;  // columns from this pair on
              if (VEC || vec_out) {
                if (room > 0) *(float2 *)(to + 8 * j) = make_float2(o[j][2 * half], o[j][2 * half + 1]);
              } else {
                if (room > 0) to[8 * j] = o[j][2 * half];
                if (room > 1) to[8 * j + 1] = o[j][2 * half + 1];
              }
            }
          }
        } else if constexpr (sizeof(T) == 2) {
          // through this warp's own rows of the query tile, 16 bytes at a time
          using Out = Tile<T, VT, 0>;
          const Out out(Q.p + 16 * warp * L::Q::kPitch, lane);
          __syncwarp();
#pragma unroll
          for (int j = 0; j < VT / 8; ++j) out.put(0, j, lane, o[j][0], o[j][1], o[j][2], o[j][3]);
          __syncwarp();
          if (VEC || vec_out) {
            constexpr int kBlocks = VT / 8, kRows = 32 / kBlocks;
            const int row = lane / kBlocks, col = lane % kBlocks * 8;
            T *to = (T *)out_to + first + row * stride + col;
#pragma unroll
            for (int i = 0; i < 16; i += kRows, to += kRows * stride)
              if (row + i < count && col < width) *(uint4 *)to = *(const uint4 *)(out.p + Out::at(row + i, col));
          } else {
            store_single<T, Out>(out.p, (T *)out_to + first, stride, count, width);
          }
        }
      }
    }

    if (c + 1 < chunks) {
      __syncwarp();  // this warp's queries have been read
      load_queries(c + 1);
    }

    // S' = lambda^rows S + (weighted K)^T V
    if (flags) {
#pragma unroll
      for (int i = 0; i < kM; ++i)
#pragma unroll
        for (int j = 0; j < kN; ++j) S[i][j][0] = S[i][j][1] = S[i][j][2] = S[i][j][3] = 0.f;
    } else {
      const float left = rows == kTile ? whole->at(c) : expf(log_decay * rows);
#pragma unroll
      for (int i = 0; i < kM; ++i)
#pragma unroll
        for (int j = 0; j < kN; ++j) scale(S[i][j], F2(left), F2(left));
    }
    cut |= flags != 0;
    const float *w = kept + rows - lag - 2 * t;
#pragma unroll 1
    for (int ks = last / 16; ks < (rows + 15) / 16; ++ks) {
      float wt[4] = {w[-16 * ks], w[-16 * ks - 1], w[-16 * ks - 8], w[-16 * ks - 9]};
      if (flags)
#pragma unroll
        for (int e = 0; e < 4; ++e) wt[e] = 16 * ks + 2 * t + (e & 1) + 8 * (e >> 1) >= last ? wt[e] : 0.f;
      A16<T> ka[kM];
#pragma unroll
      for (int i = 0; i < kM; ++i) ka[i] = K.columns_a(16 * ks, m0 + 16 * i, lane);
      B16<T> vb[kN];
#pragma unroll
      for (int j = 0; j < kN; j += 2) {
        V.columns_b(vb + j, 16 * ks, n0 + 8 * j, lane);
      }
#pragma unroll
      for (int i = 0; i < kM; ++i) {
        F2 x[4];
        ka[i].values(x);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = mul(x[e], F2(wt[2 * (e >> 1)], wt[2 * (e >> 1) + 1]));
        const Value<T, PARTS> kv(x, s.parts);
        kv.template mul<kN>(S[i], vb, s.parts);
      }
    }
    // (a state that was cut holds this chunk's own tokens only: sum them again)
    if (flags) {
#pragma unroll
      for (int i = 0; i < kM; ++i) {
        if (all_finite<kN>(S[i])) continue;
#pragma unroll
        for (int j = 0; j < kN; ++j)
          *(float4 *)S[i][j] =
              state_sums<T, L>(K.p, V.p, last, rows, m0 + 16 * i + g, n0 + 8 * j + 2 * t, kept + rows - lag);
      }
    }
    if (c + 1 < chunks) {
      __syncthreads();  // the state and the tiles have been read
      if (L::kStages == 1) load_keys(c + 1);
      if (!p.state_only) publish();
      mark(next);
    }
  }

  if (p.state_only || (s.final && piece == p.pieces - 1)) {
    float *to = p.state_only ? p.states + p.states_at[which] + ((int64_t)bh * p.pieces + piece) * kd * s.vd
                             : s.final + (int64_t)bh * kd * s.vd;
    const int top = m0 + g, left = n0 + 2 * t;
    to += top * s.vd + v0 + left;
    const bool pairs = VEC || (s.vd % 2 == 0 && (p.state_only || s.vec_final));  // (v0, left are even)
#pragma unroll
    for (int i = 0; i < kM; ++i)
#pragma unroll
      for (int j = 0; j < kN; ++j)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = 16 * i + 8 * half, col = 8 * j;
          if (top + r >= kd || left + col >= vd) continue;
          float *at = to + r * s.vd + col;
          if (pairs) *(float2 *)at = make_float2(S[i][j][2 * half], S[i][j][2 * half + 1]);
          else {
            at[0] = S[i][j][2 * half];
            if (left + col + 1 < vd) at[1] = S[i][j][2 * half + 1];
          }
        }
  }
  if (p.state_only) {
    if (v0 == 0 && tid == 0)
      p.factors[((int64_t)which * p.batch * p.heads + bh) * p.pieces + piece] = cut ? 0.f : own ? Decay(log_decay * own).at(piece) : 1.f;
    return;
  }
  // rows behind the length
  const int end = min(p.piece, p.time - s0);
  for (int pass = 0; pass < (TWIN ? 2 : 1); ++pass) {
    void *out_to = pass ? s.twin_out : s.out;
    const int width = pass ? kd : vd, across = pass ? kd : s.vd;
    for (int r = own + warp; r < end; r += kScanThreads / 32) {
      const int64_t at = (((int64_t)b * p.time + s0 + r) * p.heads + h) * across + v0;
      for (int col = lane; col < width; col += 32) {
        if (!FULL && s.out_float) ((float *)out_to)[at + col] = 0.f;
        else ((T *)out_to)[at + col] = from_float<T>(0.f);
      }
    }
  }
}

template <class T, int KT, int VT, int PARTS, int MODE, bool TWIN>
int launch_kernel(const ScanParams &p, cudaStream_t stream) {
  using L = Layout<T, KT, VT, TWIN>;
  const auto kernel = scan_kernel<T, KT, VT, PARTS, MODE, TWIN>;
  const int smem = L::kBytes;
  cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (rc != cudaSuccess) return (int)rc;
  const int64_t grid = (int64_t)p.batch * p.heads * p.pieces * p.units;
  if (grid >= 1ll << 31) return (int)cudaErrorInvalidValue;
  kernel<<<(unsigned)grid, kScanThreads, smem, stream>>>(p);
  return (int)cudaGetLastError();
}
template <class T, int KT, int VT, int PARTS, bool TWIN> int launch_mode(const ScanParams &p, int mode, cudaStream_t stream) {
  return mode == 2   ? launch_kernel<T, KT, VT, PARTS, 2, TWIN>(p, stream)
         : mode == 1 ? launch_kernel<T, KT, VT, PARTS, 1, TWIN>(p, stream)
                     : launch_kernel<T, KT, VT, PARTS, 0, TWIN>(p, stream);
}

// Scans with a twin output are launched by themselves: the choice at run time cost
// the others an eighth of their speed.
template <class T, int KT, int VT, int PARTS> int launch(const ScanParams &p, cudaStream_t stream) {
  bool full = true, vec = true, twin = false;
  for (int i = 0; i < p.scans; ++i) {
    const Scan &s = p.scan[i];
    twin = twin || s.twin_out;
    vec = vec && s.vec_q && s.vec_k && s.vec_v && s.vec_out && s.vec_final && s.vd % 2 == 0 && (!s.twin_out || (s.vec_x && s.vec_twin));
    full = full && s.kd == KT && s.vd % VT == 0 && !s.out_float && (!s.twin_out || s.vd == VT);
  }
  const int mode = !vec ? 0 : full ? 2 : 1;
  if (twin) {
    if constexpr (sizeof(T) == 2 && KT == VT) return launch_mode<T, KT, VT, PARTS, true>(p, mode, stream);
    return (int)cudaErrorInvalidValue;
  }
  return launch_mode<T, KT, VT, PARTS, false>(p, mode, stream);
}

template <class T, int VT> int launch_width(const ScanParams &p, int kt, cudaStream_t stream) {
  constexpr int kParts = std::is_same<T, __nv_bfloat16>::value ? 3 : 2;
  if (kt <= 32) return launch<T, 32, VT, kParts>(p, stream);
  if (kt <= 64) return launch<T, 64, VT, kParts>(p, stream);
  return launch<T, 128, VT, kParts>(p, stream);
}
}  // namespace scan

// CTAs that are resident on one SM.
template <class T> int scan_resident(int kt, int vt) {
  if (vt == 32)
    return kt <= 32 ? scan::Layout<T, 32, 32, false>::kResident
                    : kt <= 64 ? scan::Layout<T, 64, 32, false>::kResident : scan::Layout<T, 128, 32, false>::kResident;
  return kt <= 32 ? scan::Layout<T, 32, 64, false>::kResident
                  : kt <= 64 ? scan::Layout<T, 64, 64, false>::kResident : scan::Layout<T, 128, 64, false>::kResident;
}

// kt: the widest inner dimension; vt: 32 or 64, the slice of v.
template <class T> int scan_launch(const ScanParams &p, int kt, int vt, cudaStream_t stream) {
  return vt == 32 ? scan::launch_width<T, 32>(p, kt, stream) : scan::launch_width<T, 64>(p, kt, stream);
}

}  // namespace b200policy
