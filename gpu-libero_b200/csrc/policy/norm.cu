// Layer norm, forward and backward.  With xhat = (x - mean) * rstd and
// g = dy * weight:
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat))
//   dweight = sum over rows of dy * xhat,  dbias = sum over rows of dy
//
// Memory bound: x is read and y written once; x and dy are read and dx written
// once.  A group of G threads (8, or a CTA of 128 to 512; a warp has kernels of its
// own) holds a row in registers, R <= 16 values a thread in blocks of E (16 bytes, or
// single elements where rows are not aligned), takes the mean, then the spread around
// it and what rounding left of the mean (rows far from zero would lose it otherwise).
// The next row's loads are in flight meanwhile.  In the backward pass a thread keeps
// the same columns in every row, so that the sums over rows of dweight and dbias stay
// in its registers; CTAs leave one partial row each, which a second kernel adds in a
// fixed order.  Rows of more than 8192 are read again instead.
// 262144 rows of 1024 in bf16: 200 us forward (5.4 TB/s) and 279 us backward (5.8
// TB/s), 8 of them for the partial rows; 30011 rows of 771 floats, 1027 apart: 43 us
// (4.3 TB/s) and 59 us (4.7 TB/s).
#include <algorithm>
#include "common.cuh"

namespace {
using namespace b200policy;

constexpr int kSms = 148;
constexpr int kWideThreads = 256;
constexpr int kMostColumns = 0x7fffffff - 1024;  // column numbers a CTA's stride on are 32-bit too

template <class W> __device__ __forceinline__ float weight_at(const void *w, int i, float none) {
  return w ? to_float(((const W *)w)[i]) : none;
}

// Threads of a CTA whose groups have G.
__host__ __device__ constexpr int threads_of(int g) { return g < 128 ? 256 : g; }

// The spread around a first mean, corrected by the rest of the mean, cannot be
// negative but for rounding.
template <class A> __device__ __forceinline__ A rstd_of(A var, float eps) { return A(1) / sqrt((var > 0 ? var : 0) + eps); }

// E consecutive elements, read and written at once.
template <class T, int E> struct alignas(E * sizeof(T)) Block { T v[E]; };

// Sums of two values over a group, on all its threads, in a fixed order.  CTA
// groups pass through `part` ([2][G / 32]), whose halves alternate by `turn`, so
// that one barrier is enough.
template <int G, class V> struct Two { V x, y; };
template <int G, class V> __device__ __forceinline__ Two<G, V> group_sums(V x, V y, Two<G, V> *part, int &turn) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1) {
    x += __shfl_xor_sync(~0u, x, o);
    y += __shfl_xor_sync(~0u, y, o);
  }
  if (G <= 32) return {x, y};
  constexpr int kWarps = G / 32;
  Two<G, V> *to = part + turn * kWarps;
  turn ^= 1;
  if (threadIdx.x % 32 == 0) to[threadIdx.x / 32] = {x, y};
  __syncthreads();
  x = y = V(0);
#pragma unroll
  for (int w = 0; w < kWarps; ++w) x += to[w].x, y += to[w].y;
  return {x, y};
}

// The columns of a thread: block i of E starts at column (i * G + rank) * E.
template <class T, int E, int G, int R> struct Row {
  static constexpr int N = R / E;
  Block<T, E> b[N];
  __device__ __forceinline__ void load(const T *p, int width, int rank) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * G + rank) * E;
      if (c < width) b[i] = *(const Block<T, E> *)(p + c);
    }
  }
  __device__ __forceinline__ float at(int i, int e) const { return to_float(b[i].v[e]); }
};

// Where the group's values lie: for every block i and element e of a thread
// that is inside the row, f(i, e, column).
template <int E, int G, int R, class F> __device__ __forceinline__ void each(int width, int rank, F f) {
#pragma unroll
  for (int i = 0; i < R / E; ++i) {
    const int c = (i * G + rank) * E;
    if (c < width)
#pragma unroll
      for (int e = 0; e < E; ++e) f(i, e, c + e);
  }
}

// A: the type of a row's sums.  Groups of 8 (rows of up to 64) take 64 bits and
// recompute their statistics in the backward pass: with few elements dx is the
// small remainder (about eps / var for two) of terms of size g.
template <int G> using Sum = typename std::conditional<G == 8, double, float>::type;

template <class T, class W, int E, int G, int R>
__global__ void __launch_bounds__(threads_of(G)) forward_kernel(B200NormArgs a) {
  using A = Sum<G>;
  constexpr int kGroups = threads_of(G) / G;
  __shared__ Two<G, A> part[G > 32 ? 2 * G / 32 : 1];
  int turn = 0;
  const int rank = threadIdx.x % G, width = a.width;
  const int64_t stride = (int64_t)gridDim.x * kGroups, own = threadIdx.x / G;
  int64_t row = (int64_t)blockIdx.x * kGroups + own;
  Row<T, E, G, R> next;
  if (row < a.rows) next.load((const T *)a.x + row * a.x_row, width, rank);
  for (; row - own < a.rows; row += stride) {
    const bool on = row < a.rows;  // whole groups; every lane takes part in the sums
    const Row<T, E, G, R> x = next;
    if (row + stride < a.rows) next.load((const T *)a.x + (row + stride) * a.x_row, width, rank);
    A s = 0;
    if (on) each<E, G, R>(width, rank, [&](int i, int e, int) { s += x.at(i, e); });
    const A about = group_sums<G>(s, A(0), part, turn).x / width;  // the mean, up to rounding
    A s1 = 0, s2 = 0;
    if (on)
      each<E, G, R>(width, rank, [&](int i, int e, int) {
        const A d = x.at(i, e) - about;
        s1 += d;
        s2 += d * d;
      });
    const Two<G, A> sums = group_sums<G>(s1, s2, part, turn);
    const A off = sums.x / width, rstd = rstd_of(sums.y / width - off * off, a.eps);
    if (!on) continue;
    T *y = (T *)a.y + row * width;
#pragma unroll
    for (int i = 0; i < R / E; ++i) {
      const int c = (i * G + rank) * E;
      if (c >= width) continue;
      Block<T, E> to;
      Block<W, E> w, b;
      if (a.weight) w = *(const Block<W, E> *)((const W *)a.weight + c);
      if (a.bias) b = *(const Block<W, E> *)((const W *)a.bias + c);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float v = (float)((x.at(i, e) - about - off) * rstd);
        if (a.weight) v *= to_float(w.v[e]);
        if (a.bias) v += to_float(b.v[e]);
        to.v[e] = from_float<T>(v);
      }
      *(Block<T, E> *)(y + c) = to;
    }
    if (a.stats && rank == 0) *(float2 *)(a.stats + 2 * row) = make_float2((float)(about + off), (float)rstd);
  }
}

// A CTA's sums of one column: to its partial row, parts[CTA][dweight, dbias][width],
// or to the gradients where there is one CTA (parts is NULL).
template <class W> __device__ __forceinline__ void put_sums(const B200NormArgs &a, float *parts, int c, float dw, float db) {
  if (parts) {
    float *to = parts + (size_t)blockIdx.x * 2 * a.width;
    to[c] = dw, to[a.width + c] = db;
  } else {
    if (a.dweight) ((W *)a.dweight)[c] = from_float<W>(dw);
    if (a.dbias) ((W *)a.dbias)[c] = from_float<W>(db);
  }
}

template <class T, class W, int E, int G, int R>
__global__ void __launch_bounds__(threads_of(G)) backward_kernel(B200NormArgs a, float *parts) {
  using A = Sum<G>;
  constexpr int N = R / E, kGroups = threads_of(G) / G;
  __shared__ Two<G, A> part[G > 32 ? 2 * G / 32 : 1];
  int turn = 0;
  const int rank = threadIdx.x % G, width = a.width;
  const int64_t stride = (int64_t)gridDim.x * kGroups, own = threadIdx.x / G;
  int64_t row = (int64_t)blockIdx.x * kGroups + own;
  float dw[R] = {}, db[R] = {};
  Row<T, E, G, R> next_x, next_dy;
  float2 next_stats = {};
  auto load = [&](int64_t row) {
    next_x.load((const T *)a.x + row * a.x_row, width, rank);
    next_dy.load((const T *)a.dy + row * a.dy_row, width, rank);
    if (G != 8) next_stats = *(const float2 *)(a.stats + 2 * row);
  };
  if (row < a.rows) load(row);
  for (; row - own < a.rows; row += stride) {
    const bool on = row < a.rows;
    const Row<T, E, G, R> x = next_x, dy = next_dy;
    A mean = next_stats.x, rstd = next_stats.y;
    if (row + stride < a.rows) load(row + stride);
    if (G == 8) {
      A s = 0;
      if (on) each<E, G, R>(width, rank, [&](int i, int e, int) { s += x.at(i, e); });
      mean = group_sums<G>(s, A(0), part, turn).x / width;
      s = 0;
      if (on)
        each<E, G, R>(width, rank, [&](int i, int e, int) {
          const A d = x.at(i, e) - mean;
          s += d * d;
        });
      rstd = rstd_of(group_sums<G>(s, A(0), part, turn).x / width, a.eps);
    }
    A sg = 0, sh = 0;
    if (on) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = (i * G + rank) * E;
        if (c >= width) continue;
        Block<W, E> w;
        if (a.weight) w = *(const Block<W, E> *)((const W *)a.weight + c);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float d = dy.at(i, e);
          const A hat = (x.at(i, e) - mean) * rstd, g = a.weight ? d * A(to_float(w.v[e])) : A(d);
          sg += g;
          sh += g * hat;
          dw[i * E + e] += d * (float)hat;
          db[i * E + e] += d;
        }
      }
    }
    if (!a.dx) continue;
    const Two<G, A> sums = group_sums<G>(sg, sh, part, turn);
    if (!on) continue;
    sg = sums.x / width, sh = sums.y / width;
    T *dx = (T *)a.dx + row * width;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * G + rank) * E;
      if (c >= width) continue;
      Block<W, E> w;
      Block<T, E> to;
      if (a.weight) w = *(const Block<W, E> *)((const W *)a.weight + c);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const A d = dy.at(i, e), g = a.weight ? d * A(to_float(w.v[e])) : d;
        to.v[e] = from_float<T>((float)(rstd * (g - sg - (x.at(i, e) - mean) * rstd * sh)));
      }
      *(Block<T, E> *)(dx + c) = to;
    }
  }
  if (!a.dweight && !a.dbias) return;
  if (G > 32) {
    each<E, G, R>(width, rank, [&](int i, int e, int c) { put_sums<W>(a, parts, c, dw[i * E + e], db[i * E + e]); });
    return;
  }
  // groups of 8: a warp's by shuffles, the CTA's warps in order through shared memory
  constexpr int kColumns = G == 8 ? G * R : 1;
  __shared__ float columns[2][kColumns];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int o = 16; o >= 8; o >>= 1) {
      dw[i] += __shfl_xor_sync(~0u, dw[i], o);
      db[i] += __shfl_xor_sync(~0u, db[i], o);
    }
  for (int warp = 0; warp < threads_of(G) / 32; ++warp) {
    if (threadIdx.x / 32 == warp && threadIdx.x % 32 < G)
      each<E, G, R>(width, rank, [&](int i, int e, int c) {
        columns[0][c] = (warp ? columns[0][c] : 0.f) + dw[i * E + e];
        columns[1][c] = (warp ? columns[1][c] : 0.f) + db[i * E + e];
      });
    __syncthreads();
  }
  const int c = threadIdx.x;
  if (c < width) put_sums<W>(a, parts, c, columns[0][c], columns[1][c]);
}

// What a thread reads and writes at once, as pairs of values (one by one, ten
// instructions a value bind the rows' arithmetic): a block of E, or two single
// elements 32 columns apart.  Elements behind the row are zero.
template <class T, int E, int R> struct Unit {
  static constexpr int kCount = E == 1 ? R / 2 : R / E, kPairs = E == 1 ? 1 : E / 2;
  F2 v[kPairs];
  static __device__ __forceinline__ int column(int u) {
    return E == 1 ? 64 * u + (int)threadIdx.x % 32 : (u * 32 + (int)threadIdx.x % 32) * E;
  }
  static __device__ __forceinline__ bool in(int u, int width, int half = 0) { return column(u) + 32 * half < width; }
  template <class V> __device__ __forceinline__ void set(const Block<V, E> &b) {
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      if constexpr (std::is_same<V, __nv_bfloat16>::value && E > 1) {
        const uint32_t x = ((const uint32_t *)&b)[j];
        v[j] = F2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
      } else
        v[j] = F2(to_float(b.v[2 * j]), to_float(b.v[2 * j + 1]));
    }
  }
  // from a row in global memory
  template <class V> __device__ __forceinline__ void load(const V *row, int u, int width, float none = 0.f) {
    const int c = column(u);
    if constexpr (E == 1)
      v[0] = F2(in(u, width) ? to_float(row[c]) : none, in(u, width, 1) ? to_float(row[c + 32]) : none);
    else if (in(u, width)) set(*(const Block<V, E> *)(row + c));
    else
#pragma unroll
      for (int j = 0; j < kPairs; ++j) v[j] = F2(none);
  }
  __device__ __forceinline__ void store(T *row, int u, int width) const {
    const int c = column(u);
    if constexpr (E == 1) {
      if (in(u, width)) row[c] = from_float<T>(v[0].get().x);
      if (in(u, width, 1)) row[c + 32] = from_float<T>(v[0].get().y);
    } else {
      Block<T, E> b;
#pragma unroll
      for (int j = 0; j < kPairs; ++j) b.v[2 * j] = from_float<T>(v[j].get().x), b.v[2 * j + 1] = from_float<T>(v[j].get().y);
      if (in(u, width)) *(Block<T, E> *)(row + c) = b;
    }
  }
};

// ---- a warp to a row (of 65 to 1024) -------------------------------------------
// A CTA's reductions cost more instructions than a row of 1024 pays for (256
// threads' sums took the forward pass from 211 us to 381 at 262144 rows of bf16),
// and a warp that holds a row has no registers left for the next ones.  So rows
// arrive through a ring in shared memory, 16 bytes a copy: in blocks that each
// lane copies for itself, or, where rows start at any element, from the aligned
// address before the row (the same allocation's memory) to the row's end.
constexpr int kWarpThreads = 128;
// Stages of the ring, and its bytes of a CTA, for rows of 32 `values` elements.
__host__ __device__ constexpr int ring_stages(int values, int bytes, int tensors) { return values * bytes * tensors >= 128 ? 3 : 4; }
__host__ __device__ constexpr int ring_row(int values, int bytes, bool single) { return 32 * values * bytes + (single ? 16 : 0); }
__host__ __device__ constexpr int ring_bytes(int values, int bytes, bool single, int tensors) {
  return ring_stages(values, bytes, tensors) * tensors * ring_row(values, bytes, single) * (kWarpThreads / 32);
}
// CTAs of an SM by their registers, and also by their shared memory (of 228 KB, 1 KB
// more for each CTA; the backward pass also holds its sums); the grid is one wave of
// them.  (32-bit rows of 513 to 1024, backward: two CTAs fit; a grid of three took 72 us
// for 30011 rows of 771 instead of 59, and two stages that let three fit 64.)
__host__ __device__ constexpr int by_registers(int values, bool backward) {
  return backward ? (values == 32 ? 3 : 4) : values == 32 ? 4 : values == 16 ? 5 : 8;
}
__host__ __device__ constexpr int resident(int values, bool backward, int bytes, bool single) {
  const int held = ring_bytes(values, bytes, single, backward ? 2 : 1) + (backward ? 2 * 32 * values * 4 : 0) + 1024;
  const int fit = 228 * 1024 / held, most = by_registers(values, backward);
  return fit < most ? fit : most;
}

template <class T, int E, int R, int TENSORS> struct Ring {
  static constexpr int kStages = ring_stages(R, sizeof(T), TENSORS);
  static constexpr int kRow = ring_row(R, sizeof(T), E == 1);  // of one tensor and warp
  static constexpr int bytes() { return ring_bytes(R, sizeof(T), E == 1, TENSORS); }
  static __device__ __forceinline__ int at(int stage, int tensor) {
    return ((stage * TENSORS + tensor) * (kWarpThreads / 32) + threadIdx.x / 32) * kRow;
  }
  static __device__ __forceinline__ void copy(unsigned char *to, const void *from, int size) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from),
                 "r"(size)
                 : "memory");
  }
  static __device__ __forceinline__ void fetch(unsigned char *ring, int stage, int tensor, const T *row, int width) {
    const int lane = threadIdx.x % 32;
    ring += at(stage, tensor);
    if (E == 1) {
      const int skip = (int)((uintptr_t)row & 15), size = skip + width * (int)sizeof(T);
      const unsigned char *from = (const unsigned char *)row - skip;
#pragma unroll
      for (int i = 0; i < (kRow + 511) / 512; ++i) {
        const int c = (i * 32 + lane) * 16;
        if (c < size) copy(ring + c, from + c, min(16, size - c));
      }
    } else {
#pragma unroll
      for (int i = 0; i < R / E; ++i) {
        const int c = (i * 32 + lane) * E;
        if (c < width) copy(ring + c * sizeof(T), row + c, 16);
      }
    }
  }
  static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  static __device__ __forceinline__ void wait() {  // for the oldest of kStages groups
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    if (E == 1) __syncwarp();
  }
  static __device__ __forceinline__ void done() {  // before a stage that other lanes read is fetched again
    if (E == 1) __syncwarp();
  }
  // block u of a fetched row, as it is (zero behind the row)
  static __device__ __forceinline__ Block<T, E> block(const unsigned char *ring, int stage, int tensor, int u, int width) {
    Block<T, E> b = {};
    const int c = Unit<T, E, R>::column(u);
    if (c < width) b = *(const Block<T, E> *)(ring + at(stage, tensor) + c * sizeof(T));
    return b;
  }
  // unit u of a fetched row
  static __device__ __forceinline__ Unit<T, E, R> take(const unsigned char *ring, int stage, int tensor, const T *row, int u,
                                                       int width) {
    Unit<T, E, R> x;
    x.load((const T *)(ring + at(stage, tensor) + (E == 1 ? (uintptr_t)row & 15 : 0)), u, width);
    return x;
  }
};

template <class T, class W, int E, int R>
__global__ void __launch_bounds__(kWarpThreads, resident(R, false, sizeof(T), E == 1)) forward_warps(B200NormArgs a) {
  using Rows = Ring<T, E, R, 1>;
  extern __shared__ __align__(16) unsigned char ring[];
  const int rank = threadIdx.x % 32, width = a.width;
  const int64_t stride = (int64_t)gridDim.x * (kWarpThreads / 32);
  const int64_t start = (int64_t)blockIdx.x * (kWarpThreads / 32) + threadIdx.x / 32;
  const T *x0 = (const T *)a.x;
#pragma unroll
  for (int i = 0; i < Rows::kStages; ++i) {
    if (start + i * stride < a.rows) Rows::fetch(ring, i, 0, x0 + (start + i * stride) * a.x_row, width);
    Rows::commit();
  }
  using U = Unit<T, E, R>;
  U w[U::kCount], b[U::kCount];
#pragma unroll
  for (int u = 0; u < U::kCount; ++u) {
    if (a.weight) w[u].load((const W *)a.weight, u, width);
    else
#pragma unroll
      for (int j = 0; j < U::kPairs; ++j) w[u].v[j] = F2(1.f);
    if (a.bias) b[u].load((const W *)a.bias, u, width);
  }
  const float share = 1.f / width;
  int stage = 0;
  for (int64_t row = start; row < a.rows; row += stride) {
    const T *from = x0 + row * a.x_row;
    Rows::wait();
    auto refill = [&] {
      Rows::done();
      if (row + Rows::kStages * stride < a.rows)
        Rows::fetch(ring, stage, 0, x0 + (row + Rows::kStages * stride) * a.x_row, width);
      Rows::commit();
      stage = stage + 1 == Rows::kStages ? 0 : stage + 1;
    };
    // blocks are held as they are and widened in each of the three passes; single
    // elements are read from the ring three times
    Block<T, E> held[E > 1 ? R / E : 1];
    if constexpr (E > 1) {
#pragma unroll
      for (int u = 0; u < U::kCount; ++u) held[u] = Rows::block(ring, stage, 0, u, width);
      refill();
    }
    auto take = [&](int u) {
      if constexpr (E == 1) return Rows::take(ring, stage, 0, from, u, width);
      else {
        U x;
        x.set(held[u]);
        return x;
      }
    };
    F2 s;
#pragma unroll
    for (int u = 0; u < U::kCount; ++u) {
      const U x = take(u);
#pragma unroll
      for (int j = 0; j < U::kPairs; ++j) s = add(s, x.v[j]);
    }
    const float about = warp_sum(s.sum()) * share;  // the mean, up to rounding
    F2 s1, s2;
#pragma unroll
    for (int u = 0; u < U::kCount; ++u) {
      const U x = take(u);
#pragma unroll
      for (int j = 0; j < U::kPairs; ++j) {
        F2 d = add(x.v[j], F2(-about));
        if constexpr (E == 1) d = F2(x.in(u, width) ? d.get().x : 0.f, x.in(u, width, 1) ? d.get().y : 0.f);
        else if (!x.in(u, width)) continue;
        s1 = add(s1, d);
        s2 = fma(d, d, s2);
      }
    }
    const float off = warp_sum(s1.sum()) * share, rstd = rstd_of(warp_sum(s2.sum()) * share - off * off, a.eps);
#pragma unroll
    for (int u = 0; u < U::kCount; ++u) {
      U x = take(u);
#pragma unroll
      for (int j = 0; j < U::kPairs; ++j)
        x.v[j] = fma(mul(add(add(x.v[j], F2(-about)), F2(-off)), F2(rstd)), w[u].v[j], b[u].v[j]);
      x.store((T *)a.y + row * width, u, width);
    }
    if (E == 1) refill();
    if (a.stats && rank == 0) *(float2 *)(a.stats + 2 * row) = make_float2(about + off, rstd);
  }
}

template <class T, class W, int E, int R>
__global__ void __launch_bounds__(kWarpThreads, resident(R, true, sizeof(T), E == 1)) backward_warps(B200NormArgs a, float *parts) {
  using Rows = Ring<T, E, R, 2>;
  extern __shared__ __align__(16) unsigned char ring[];
  const int width = a.width;
  const int64_t stride = (int64_t)gridDim.x * (kWarpThreads / 32);
  const int64_t start = (int64_t)blockIdx.x * (kWarpThreads / 32) + threadIdx.x / 32;
  const T *x0 = (const T *)a.x, *dy0 = (const T *)a.dy;
#pragma unroll
  for (int i = 0; i < Rows::kStages; ++i) {
    if (start + i * stride < a.rows) {
      Rows::fetch(ring, i, 0, x0 + (start + i * stride) * a.x_row, width);
      Rows::fetch(ring, i, 1, dy0 + (start + i * stride) * a.dy_row, width);
    }
    Rows::commit();
  }
  using U = Unit<T, E, R>;
  U w[U::kCount], dw[U::kCount], db[U::kCount];
#pragma unroll
  for (int u = 0; u < U::kCount; ++u) {
    if (a.weight) w[u].load((const W *)a.weight, u, width);
    else
#pragma unroll
      for (int j = 0; j < U::kPairs; ++j) w[u].v[j] = F2(1.f);
  }
  const float share = 1.f / width;
  float2 stats = start < a.rows ? *(const float2 *)(a.stats + 2 * start) : make_float2(0.f, 0.f);
  int stage = 0;
  for (int64_t row = start; row < a.rows; row += stride) {
    Rows::wait();
    const F2 less(-stats.x), rstd(stats.y);
    if (row + stride < a.rows) stats = *(const float2 *)(a.stats + 2 * (row + stride));
    F2 sg, sh;
    // both passes read the row from the ring: the sums over rows leave no room for it
#pragma unroll
    for (int u = 0; u < U::kCount; ++u) {
      // zero behind the row: no sum takes anything from dy = 0
      const U x = Rows::take(ring, stage, 0, x0 + row * a.x_row, u, width);
      const U dy = Rows::take(ring, stage, 1, dy0 + row * a.dy_row, u, width);
#pragma unroll
      for (int j = 0; j < U::kPairs; ++j) {
        const F2 d = dy.v[j], hat = mul(add(x.v[j], less), rstd), g = mul(d, w[u].v[j]);
        sg = add(sg, g);
        sh = fma(g, hat, sh);
        dw[u].v[j] = fma(d, hat, dw[u].v[j]);
        db[u].v[j] = add(db[u].v[j], d);
      }
    }
    if (a.dx) {
      const F2 mg(-warp_sum(sg.sum()) * share), mh(-warp_sum(sh.sum()) * share);
#pragma unroll
      for (int u = 0; u < U::kCount; ++u) {
        U x = Rows::take(ring, stage, 0, x0 + row * a.x_row, u, width);
        const U dy = Rows::take(ring, stage, 1, dy0 + row * a.dy_row, u, width);
#pragma unroll
        for (int j = 0; j < U::kPairs; ++j) {
          const F2 hat = mul(add(x.v[j], less), rstd), g = mul(dy.v[j], w[u].v[j]);
          x.v[j] = mul(add(fma(hat, mh, g), mg), rstd);
        }
        x.store((T *)a.dx + row * width, u, width);
      }
    }
    Rows::done();
    if (row + Rows::kStages * stride < a.rows) {
      Rows::fetch(ring, stage, 0, x0 + (row + Rows::kStages * stride) * a.x_row, width);
      Rows::fetch(ring, stage, 1, dy0 + (row + Rows::kStages * stride) * a.dy_row, width);
    }
    Rows::commit();
    stage = stage + 1 == Rows::kStages ? 0 : stage + 1;
  }
  if (!a.dweight && !a.dbias) return;
  // the CTA's warps, in order
  __shared__ float columns[2][32 * R];
  for (int warp = 0; warp < kWarpThreads / 32; ++warp) {
    if (threadIdx.x / 32 == warp)
#pragma unroll
      for (int u = 0; u < U::kCount; ++u)
#pragma unroll
        for (int j = 0; j < U::kPairs; ++j)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int c = U::column(u) + (E == 1 ? 32 * half : 2 * j + half);
            const float2 x = dw[u].v[j].get(), y = db[u].v[j].get();
            columns[0][c] = (warp ? columns[0][c] : 0.f) + (half ? x.y : x.x);
            columns[1][c] = (warp ? columns[1][c] : 0.f) + (half ? y.y : y.x);
          }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < width; c += kWarpThreads) put_sums<W>(a, parts, c, columns[0][c], columns[1][c]);
}

// ---- rows wider than a CTA's registers: read again for every sum --------------
template <class T, class W> __global__ void __launch_bounds__(kWideThreads) forward_wide(B200NormArgs a) {
  __shared__ float part[32];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = (const T *)a.x + row * a.x_row;
    T *y = (T *)a.y + row * a.width;
    float s = 0.f;
    for (int i = threadIdx.x; i < a.width; i += kWideThreads) s += to_float(x[i]);
    const float about = block_sum(s, part) / a.width;
    float s1 = 0.f, s2 = 0.f;
    for (int i = threadIdx.x; i < a.width; i += kWideThreads) {
      const float d = to_float(x[i]) - about;
      s1 += d;
      s2 += d * d;
    }
    const float off = block_sum(s1, part) / a.width, mean = about + off;
    const float rstd = rstd_of(block_sum(s2, part) / a.width - off * off, a.eps);
    for (int i = threadIdx.x; i < a.width; i += kWideThreads)
      y[i] = from_float<T>((to_float(x[i]) - about - off) * rstd * weight_at<W>(a.weight, i, 1.f) + weight_at<W>(a.bias, i, 0.f));
    if (a.stats && threadIdx.x == 0) a.stats[2 * row] = mean, a.stats[2 * row + 1] = rstd;
  }
}

template <class T, class W> __global__ void __launch_bounds__(kWideThreads) backward_wide(B200NormArgs a) {
  __shared__ float part[32];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = (const T *)a.x + row * a.x_row, *dy = (const T *)a.dy + row * a.dy_row;
    T *dx = (T *)a.dx + row * a.width;
    const float mean = a.stats[2 * row], rstd = a.stats[2 * row + 1];
    float sg = 0.f, sh = 0.f;
    for (int i = threadIdx.x; i < a.width; i += kWideThreads) {
      const float g = to_float(dy[i]) * weight_at<W>(a.weight, i, 1.f);
      sg += g;
      sh += g * (to_float(x[i]) - mean) * rstd;
    }
    sg = block_sum(sg, part) / a.width;
    sh = block_sum(sh, part) / a.width;
    for (int i = threadIdx.x; i < a.width; i += kWideThreads) {
      const float g = to_float(dy[i]) * weight_at<W>(a.weight, i, 1.f);
      dx[i] = from_float<T>(rstd * (g - sg - (to_float(x[i]) - mean) * rstd * sh));
    }
  }
}

// The p-th range of rows of one block of columns.
template <class T> __global__ void __launch_bounds__(kWideThreads) columns_wide(B200NormArgs a, float *parts) {
  const int i = blockIdx.x * kWideThreads + threadIdx.x;
  const int64_t low = a.rows * blockIdx.y / gridDim.y, high = a.rows * (blockIdx.y + 1) / gridDim.y;
  if (i >= a.width) return;
  float sw = 0.f, sb = 0.f;
  for (int64_t row = low; row < high; ++row) {
    const float dy = to_float(((const T *)a.dy)[row * a.dy_row + i]);
    const float x = to_float(((const T *)a.x)[row * a.x_row + i]);
    sw += dy * (x - a.stats[2 * row]) * a.stats[2 * row + 1];
    sb += dy;
  }
  parts[(blockIdx.y * 2) * (size_t)a.width + i] = sw;
  parts[(blockIdx.y * 2 + 1) * (size_t)a.width + i] = sb;
}

// dweight and dbias from the CTAs' partial rows: 32 columns a CTA, a range of
// partial rows to each of its 32 warps.
template <class W> __global__ void __launch_bounds__(1024) totals_kernel(B200NormArgs a, const float *parts, int count) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, which = blockIdx.y;
  float s = 0.f;
  if (c < a.width)
#pragma unroll 8
    for (int p = warp; p < count; p += 32) s += parts[((size_t)p * 2 + which) * a.width + c];
  part[warp][lane] = s;
  __syncthreads();
  s = warp_sum(part[lane][warp]);  // a column to each warp
  const int column = blockIdx.x * 32 + warp;
  W *to = (W *)(which ? a.dbias : a.dweight);
  if (to && lane == 0 && column < a.width) to[column] = from_float<W>(s);
}

bool args_ok(const B200NormArgs *a) {
  return a && dtype_ok(a->dtype) && (a->weight_dtype == a->dtype || a->weight_dtype == B200_FP32) && a->rows >= 0 &&
         a->rows < (1ll << 31) && a->width > 0 && a->width <= kMostColumns && (uintptr_t)a->stats % 8 == 0;
}

// Calls f with values of the row's and the weight's element types.
template <class F> int by_types(const B200NormArgs *a, F f) {
  return by_dtype(a->dtype, [&](auto type) {
    return a->weight_dtype == a->dtype ? f(type, type) : f(type, float());
  });
}

bool blocks_of(const void *p, int64_t row, int width, int e, size_t bytes) {
  return (uintptr_t)p % (e * bytes) == 0 && row % e == 0 && width % e == 0;
}

// What a launch takes.
struct Plan {
  int group, values, grid;  // group 0: wider than a CTA's registers
  int block;                // elements that are read and written at once
  bool single;              // one CTA's partial row is the sum
};

Plan plan_of(const B200NormArgs *a, bool backward) {
  Plan p{};
  const size_t bytes = element_bytes(a->dtype), wbytes = element_bytes(a->weight_dtype);
  const int e = (int)(16 / bytes);
  const bool blocks = blocks_of(a->x, a->x_row, a->width, e, bytes) &&
                      blocks_of(backward ? (const void *)a->dy : a->y, backward ? a->dy_row : 0, a->width, e, bytes) &&
                      (uintptr_t)(backward ? a->dx : nullptr) % 16 == 0 && (uintptr_t)a->weight % (e * wbytes) == 0 &&
                      (uintptr_t)(backward ? nullptr : a->bias) % (e * wbytes) == 0;
  p.block = blocks ? e : 1;
  p.group = a->width <= 64 ? 8 : a->width <= 1024 ? 32 : a->width <= 2048 ? 128 : a->width <= 4096 ? 256
                : a->width <= 8192 ? 512 : 0;
  p.values = p.group == 32 ? (a->width <= 256 ? 8 : a->width <= 512 ? 16 : 32) : a->width <= p.group * 8 ? 8 : 16;
  // Enough CTAs to fill the SMs; in the backward pass no more than are resident
  // at once, as each leaves a partial row.
  const int groups = p.group == 32 ? kWarpThreads / 32 : p.group ? threads_of(p.group) / p.group : 1;
  const int most = p.group == 32 ? resident(p.values, backward, (int)bytes, !blocks)
                   : !backward   ? 16
                   : p.group == 128 ? 6 : p.group == 512 ? 2 : 3;
  // a handful of rows: one CTA's sums are the totals, which saves a launch
  p.single = backward && p.group && a->rows <= 4 * groups;
  p.grid = p.single ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>((a->rows + groups - 1) / groups, kSms * most));
  return p;
}

// Calls f with the kernel's (E, G, R) as integral constants.
template <int V> using Int = std::integral_constant<int, V>;
template <class T, class F> int by_plan(const Plan &p, F f) {
  auto group = [&](auto e) {
    auto values = [&](auto g) { return p.values == 8 ? f(e, g, Int<8>()) : f(e, g, Int<16>()); };
    switch (p.group) {
      case 8: return f(e, Int<8>(), Int<8>());
      case 128: return values(Int<128>());
      case 256: return values(Int<256>());
      default: return values(Int<512>());
    }
  };
  auto warp = [&](auto e) {
    return p.values == 8 ? f(e, Int<32>(), Int<8>()) : p.values == 16 ? f(e, Int<32>(), Int<16>()) : f(e, Int<32>(), Int<32>());
  };
  constexpr int kBlock = 16 / sizeof(T);
  if (p.group == 32) {
    if (p.block == kBlock) return warp(Int<kBlock>());
    return warp(Int<1>());
  }
  return p.block == kBlock ? group(Int<kBlock>()) : group(Int<1>());
}

template <class K> int ring_smem(K kernel, int bytes) {
  return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
}  // namespace

extern "C" {
size_t b200policy_norm_bytes(void) { return sizeof(B200NormArgs); }

size_t b200policy_norm_workspace(const B200NormArgs *a) {
  if (!args_ok(a) || (!a->dweight && !a->dbias) || plan_of(a, true).single) return 0;
  return (size_t)plan_of(a, true).grid * 2 * a->width * sizeof(float);
}

int b200policy_norm_forward(const B200NormArgs *a, void *stream) {
  if (!args_ok(a)) return (int)cudaErrorInvalidValue;
  if (a->rows == 0) return 0;
  if (!a->x || !a->y) return (int)cudaErrorInvalidValue;
  const Plan p = plan_of(a, false);
  return by_types(a, [&](auto type, auto weight) {
    using T = decltype(type);
    using W = decltype(weight);
    const cudaStream_t s = (cudaStream_t)stream;
    if (!p.group) forward_wide<T, W><<<p.grid, kWideThreads, 0, s>>>(*a);
    else
      by_plan<T>(p, [&](auto e, auto g, auto r) {
        constexpr int E = e.value, G = g.value, R = r.value;
        if constexpr (G == 32) {
          constexpr int smem = Ring<T, E, R, 1>::bytes();
          if (int rc = ring_smem(forward_warps<T, W, E, R>, smem)) return rc;
          forward_warps<T, W, E, R><<<p.grid, kWarpThreads, smem, s>>>(*a);
        } else {
          forward_kernel<T, W, E, G, R><<<p.grid, threads_of(G), 0, s>>>(*a);
        }
        return 0;
      });
    return (int)cudaGetLastError();
  });
}

int b200policy_norm_backward(const B200NormArgs *a, void *stream) {
  if (!args_ok(a) || (a->rows && !(a->x && a->dy && a->stats))) return (int)cudaErrorInvalidValue;
  if (b200policy_norm_workspace(a) && (!a->workspace || (uintptr_t)a->workspace % 16)) return (int)cudaErrorInvalidValue;
  const Plan p = plan_of(a, true);
  return by_types(a, [&](auto type, auto weight) {
    using T = decltype(type);
    using W = decltype(weight);
    const cudaStream_t s = (cudaStream_t)stream;
    const bool sums = a->dweight || a->dbias;
    float *parts = sums && !p.single ? (float *)a->workspace : nullptr;
    if (p.group) {
      by_plan<T>(p, [&](auto e, auto g, auto r) {
        constexpr int E = e.value, G = g.value, R = r.value;
        if constexpr (G == 32) {
          constexpr int smem = Ring<T, E, R, 2>::bytes();
          if (int rc = ring_smem(backward_warps<T, W, E, R>, smem)) return rc;
          backward_warps<T, W, E, R><<<p.grid, kWarpThreads, smem, s>>>(*a, parts);
        } else {
          backward_kernel<T, W, E, G, R><<<p.grid, threads_of(G), 0, s>>>(*a, parts);
        }
        return 0;
      });
    } else {
      if (a->dx && a->rows) backward_wide<T, W><<<p.grid, kWideThreads, 0, s>>>(*a);
      if (parts) columns_wide<T><<<dim3((a->width + kWideThreads - 1) / kWideThreads, p.grid), kWideThreads, 0, s>>>(*a, parts);
    }
    if (parts) totals_kernel<W><<<dim3((a->width + 31) / 32, 2), 1024, 0, s>>>(*a, parts, p.grid);
    return (int)cudaGetLastError();
  });
}
}
