// The trajectory form of decay attention in bf16 on the fifth-generation tensor
// cores: the scan of attention_scan.cuh in chunks of 128 tokens, with the
// operands in shared memory and the products in tensor memory.
//
// One thread issues a chunk's products; the 256 threads only weigh, round and move
// values, two of them to a token's row, each half of its columns:
//   A  = Q K^T                     [128, 128]
//   B  = Q S                       [128, 64]
//   D  = K^T (weighted V)          [128, 64 for each term]
//   P  = weighted A in bf16
//   C  = P V                       [128, 64]
//   out = out weight * B + C,  S = lambda^rows S + D (in registers, 32 bits)
// The weighted V is three bf16 terms (two where no state leaves), as the weighted
// K there; one product of N = 192 takes all three.  The threads split V while A and
// B are computed, make P while D is, and take B home and update S while C is.  The
// next chunk's loads fly all the while: two buffers of Q, K and V, and so one CTA an
// SM (226 KB).
//
// What bounds it is the chain of a chunk's steps, 7600 cycles for 128 tokens of a
// slice, of which the tensor cores work 2300 (8 heads of 128 and 32771 tokens: 127 us
// for the outputs, 74 us before them for the pieces' states).  Heads of 64 and less
// keep the warp-level kernel: there a chunk is half the work and the chain as long.
//
// Every wait on a barrier is bounded: when one runs out, the CTA writes its call's
// number into the status word, and stops after freeing its tensor memory; the call's
// other CTAs stop when they see the number, those of other calls do not.
#include "attention_scan.h"
#include "common.cuh"

namespace b200policy {
namespace tc {

constexpr int kRows = 128, kThreads = 256, kVt = 64, kWidth = 128;
constexpr int kSub = kRows * 128;  // bytes of 128 rows of 64 elements
using bf16 = __nv_bfloat16;

// Shared memory: two buffers of Q, K (two parts of 64 columns each) and V; the
// weighted V's terms; S; tables.
constexpr int kQ = 0, kK = 2 * kSub, kV = 4 * kSub, kBuffer = 5 * kSub, kW = 2 * kBuffer, kS = kW + 3 * kSub;
constexpr int kTables = kS + kWidth * 128;
// floats: into[0..128], within[-32..128], kept[0..128], fall[32]
constexpr int kInto = 0, kWithin = 132 + 32, kKept = kWithin + 132, kFall = kKept + 132, kFloats = kFall + 32;
constexpr int kBars = kTables + kFloats * 4, kMarks = kBars + 3 * 8, kTmem = kMarks + 4 * 4;
constexpr int kBytes = kTmem + 4;
static_assert(kBytes <= 227 * 1024, "shared memory of a CTA");
// Columns of tensor memory.
constexpr int kColumns = 512, kColA = 0, kColB = 128, kColC = 192, kColD = 256, kColP = 448;

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// Descriptor of a 128-byte-swizzled operand whose 8-row groups are 1024 bytes
// apart; lead: bytes between 64-element parts of the contiguous dimension.
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t lead) {
  return (uint64_t)((at & 0x3ffff) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// bf16 operands, 32-bit sums; whether A and B are contiguous along M and N.
__host__ __device__ __forceinline__ constexpr uint32_t instruction(int n, bool a_rows, bool b_rows) {
  return 1u << 4 | 1u << 7 | 1u << 10 | (uint32_t)a_rows << 15 | (uint32_t)b_rows << 16 | (uint32_t)(n / 8) << 17 |
         (uint32_t)(128 / 16) << 24;
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t what, bool add) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(what), "r"((uint32_t)add)
               : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t what, bool add) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(what), "r"((uint32_t)add)
               : "memory");
}
// Up to eight steps of depth 16, unrolled: a product is issued every 50 to 100
// cycles so, and every 190 where a loop computes its operands.  The operands
// advance by A and B (in 16-byte units).
template <int A, int B> __device__ __forceinline__ void issue(uint32_t d, uint64_t a, uint64_t b, uint32_t what, int steps, bool add) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < steps) mma(d, a + i * A, b + i * B, what, add || i > 0);
}
template <int B> __device__ __forceinline__ void issue_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t what, int steps) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < steps) mma_tmem(d, a + i * 8, b + i * B, what, i > 0);
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint64_t nanoseconds() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
// True when the barrier's phase is done; false when a second has passed.
__device__ __forceinline__ bool wait(uint32_t bar, int parity) {
  auto done = [&] {
    uint32_t r;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(r)
                 : "r"(bar), "r"(parity), "r"(1000)
                 : "memory");
    return r != 0;
  };
  bool ok = done();
  if (!ok) {
    const uint64_t start = nanoseconds();
#pragma unroll 1
    for (int i = 0; i < 1 << 24 && !ok && nanoseconds() - start < 1000000000ull; ++i) ok = done();
  }
  __syncwarp();  // the tensor-memory loads behind a wait are the whole warp's
  return ok;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

#define B200_X32(m) m(0), m(1), m(2), m(3), m(4), m(5), m(6), m(7), m(8), m(9), m(10), m(11), m(12), m(13), m(14), m(15), m(16), \
    m(17), m(18), m(19), m(20), m(21), m(22), m(23), m(24), m(25), m(26), m(27), m(28), m(29), m(30), m(31)
#define B200_X16(m) m(0), m(1), m(2), m(3), m(4), m(5), m(6), m(7), m(8), m(9), m(10), m(11), m(12), m(13), m(14), m(15)
// 32 columns of the lane's row.
__device__ __forceinline__ void load32(float *x, uint32_t from) {
#define B200_OUT(i) "=f"(x[i])
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
      "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : B200_X32(B200_OUT)
      : "r"(from));
#undef B200_OUT
}
__device__ __forceinline__ void load16(float *x, uint32_t from) {
#define B200_OUT(i) "=f"(x[i])
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : B200_X16(B200_OUT)
               : "r"(from));
#undef B200_OUT
}
template <int N> __device__ __forceinline__ void load_wait(float *x) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  // nothing that uses x may move before the wait
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(x[i]));
}
__device__ __forceinline__ void store8(uint32_t to, const uint32_t *x) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(x[0]), "r"(x[1]), "r"(x[2]),
               "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]), "r"(to)
               : "memory");
}
__device__ __forceinline__ void store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&p);
}
// element (row, col) of rows of 64 elements, 16-byte blocks permuted by the row
__device__ __forceinline__ int at(int row, int col) { return row * 64 + ((((col >> 3) ^ (row & 7)) << 3) | (col & 7)); }
__device__ __forceinline__ uint4 *block_of(unsigned char *tile, int row, int block) {
  return (uint4 *)(tile + row * 128 + ((block ^ (row & 7)) << 4));
}

// 64-column parts of rows of `stride` from `base`, the first `rows` of them and
// the first `width` columns; the rest is zero.  16 bytes a copy.
template <int PARTS> struct Rows {
  const bf16 *base;
  int64_t stride;
  int width;
  __device__ __forceinline__ void load(unsigned char *tile, int chunk, int rows) const {
    const int row = threadIdx.x / 8, block = threadIdx.x % 8;
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      const int col = part * 64 + block * 8;
      const bf16 *from = base + ((int64_t)chunk * kRows + row) * stride + (col < width ? col : 0);
      const uint32_t to = smem_addr(block_of(tile + part * kSub, row, block));
      constexpr int kAtOnce = kThreads / 8;
      if (rows == kRows && col < width) {
#pragma unroll
        for (int i = 0; i < kRows / kAtOnce; ++i, from += kAtOnce * stride)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * kAtOnce * 128), "l"(from) : "memory");
      } else {
#pragma unroll 1
        for (int i = 0; i < kRows / kAtOnce; ++i, from += kAtOnce * stride) {
          const bool take = col < width && row + kAtOnce * i < rows;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + i * kAtOnce * 128), "l"(take ? from : base),
                       "r"(take ? 16 : 0)
                       : "memory");
        }
      }
    }
  }
};

// Sums of a row, or of a row of the state, over their own tokens alone, where a
// product of zero and something that is not finite has spoilt them.
__device__ __noinline__ float row_sum(const bf16 *q, const bf16 *k, const bf16 *v, const bf16 *S, int i, int col, int low,
                                      bool carried, int kd, float into, const float *within) {
  float x = 0.f;
  if (carried) {
#pragma unroll 1
    for (int d = 0; d < kd; ++d) x += to_float(q[d / 64 * (kSub / 2) + at(i, d % 64)]) * to_float(S[at(d, col)]);
    x *= into;
  }
#pragma unroll 1
  for (int j = low; j <= i; ++j) {
    float dot = 0.f;
#pragma unroll 1
    for (int d = 0; d < kd; ++d)
      dot += to_float(q[d / 64 * (kSub / 2) + at(i, d % 64)]) * to_float(k[d / 64 * (kSub / 2) + at(j, d % 64)]);
    x += dot * within[i - j] * to_float(v[at(j, col)]);
  }
  return x;
}
__device__ __noinline__ float state_sum(const bf16 *k, const bf16 *v, int low, int rows, int r, int col, const float *kept) {
  float x = 0.f;
#pragma unroll 1
  for (int j = low; j < rows; ++j)
    x += to_float(k[r / 64 * (kSub / 2) + at(j, r % 64)]) * kept[-j] * to_float(v[at(j, col)]);
  return x;
}

__global__ void __launch_bounds__(kThreads, 1) scan_kernel(const __grid_constant__ ScanParams p, int *status, int call) {
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *W = smem + kW, *Ss = smem + kS;
  float *tables = (float *)(smem + kTables);
  float *into = tables + kInto, *within = tables + kWithin, *kept = tables + kKept, *fall = tables + kFall;
  unsigned *marks = (unsigned *)(smem + kMarks);
  const uint32_t bars = smem_addr(smem + kBars);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // a token's row, which is the lane of tensor memory, and the half of its columns
  const int part = warp & 3, half = warp >> 2, token = part * 32 + lane;

  // a wait has run out, here or in another CTA of this call: its outputs are void
  bool lost = threadIdx.x == 0 && *(volatile int *)status == call;
  int unit = blockIdx.x % p.units, which = 0;
  while (unit >= p.scan[which].slices) unit -= p.scan[which++].slices;
  const Scan &s = p.scan[which];
  const int v0 = unit * kVt, kd = s.kd, vd = min(kVt, s.vd - v0);
  const int rest = blockIdx.x / p.units, piece = rest % p.pieces, bh = rest / p.pieces;
  const int b = bh / p.heads, h = bh % p.heads, shared_h = h / p.group;
  const int n = p.lengths ? min(max(p.lengths[b], 0), p.time) : p.time;
  const int s0 = piece * p.piece, own = min(max(n - s0, 0), p.piece);
  const int chunks = (own + kRows - 1) / kRows;
  const int step = s.reverse ? -1 : 1, lag = s.reverse ? 0 : 1;
  const int origin = s.reverse ? n - 1 - s0 : s0;
  const Rows<2> load_q{
      (const bf16 *)s.q + b * s.q_batch + (s.q_shared ? shared_h : h) * s.q_head + origin * s.q_time, step * s.q_time, kd};
  const Rows<2> load_k{
      (const bf16 *)s.k + b * s.k_batch + (s.k_shared ? shared_h : h) * s.k_head + origin * s.k_time, step * s.k_time, kd};
  const Rows<1> load_v{
      (const bf16 *)s.v + b * s.v_batch + (s.v_shared ? shared_h : h) * s.v_head + origin * s.v_time + v0, step * s.v_time, vd};
  auto load = [&](int c) {
    const int rows = min(kRows, own - c * kRows);
    unsigned char *to = smem + (c & 1) * kBuffer;
    if (!p.state_only) load_q.load(to + kQ, c, rows);
    load_k.load(to + kK, c, rows);
    load_v.load(to + kV, c, rows);
  };
  auto starts = [&](int c) {
    const int i = c * kRows + tid;
    return p.first && tid < kRows && i < own && p.first[b * p.first_batch + (int64_t)(origin + step * i) * p.first_time];
  };
  bool next = chunks && starts(0);
  if (chunks) load(0);

  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(smem + kTmem)), "n"(kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid == 0) {
    for (int i = 0; i < 3; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bars + 8 * i) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const float log_decay = p.log_decay[h];
  const Decay whole(log_decay * kRows);
  for (int m = tid - 32; m <= kRows; m += kThreads) {
    const float x = m > 0 ? expf(log_decay * m) : m == 0 ? 1.f : 0.f;
    within[m] = x * s.pair_scale * s.out_scale;
    if (m >= 0) into[m] = x * s.out_scale;
    if (m >= 0) kept[m] = x * s.pair_scale;
    if (m >= 0 && m < 32) fall[31 - m] = x;
  }

  // S: half a row
  constexpr int kN = 32;
  const int row = token, col0 = half * 32;
  float S[kN];
  {
    const float *init = s.init;
    int64_t across = s.init_row, along = s.init_col;
    if (init) init += (int64_t)bh * kd * s.vd;
    if (p.state_only) init = nullptr;
    else if (p.pieces > 1) {
      init = p.states + p.states_at[which] + ((int64_t)bh * p.pieces + piece) * kd * s.vd;
      across = s.vd, along = 1;
    }
    if (init) init += row * across + (v0 + col0) * along;
    if (init && row < kd && along == 1 && vd == kVt && (uintptr_t)init % 16 == 0) {
#pragma unroll
      for (int j = 0; j < kN; j += 4) {
        const float4 x = *(const float4 *)(init + j);
        S[j] = x.x, S[j + 1] = x.y, S[j + 2] = x.z, S[j + 3] = x.w;
      }
    } else if (init && row < kd) {
#pragma unroll
      for (int j = 0; j < kN; ++j, init += along) S[j] = col0 + j < vd ? *init : 0.f;
    } else {
#pragma unroll
      for (int j = 0; j < kN; ++j) S[j] = 0.f;
    }
  }
  auto publish = [&] {  // S in bf16, [KT][64]
#pragma unroll
    for (int j = 0; j < kN / 8; ++j)
      *block_of(Ss, row, col0 / 8 + j) = make_uint4(pack(S[8 * j], S[8 * j + 1]), pack(S[8 * j + 2], S[8 * j + 3]),
                                                    pack(S[8 * j + 4], S[8 * j + 5]), pack(S[8 * j + 6], S[8 * j + 7]));
  };
  auto mark = [&](bool start) {
    const unsigned m = __ballot_sync(~0u, start);
    if (lane == 0 && warp < 4) marks[warp] = m;
  };
  mark(next);
  if (!p.state_only) publish();

  uint32_t tmem = 0;
  bool cut = false;
#pragma unroll 1
  for (int c = 0; c < chunks; ++c) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    fence_smem();
    fence_before();
    lost = __syncthreads_or(lost);
    fence_after();
    if (lost) break;
    tmem = *(const uint32_t *)(smem + kTmem);
    const uint32_t mine = tmem + ((uint32_t)part << 21);  // lanes 32 part and on
    const int rows = min(kRows, own - c * kRows), steps = (rows + 15) / 16;
    unsigned char *Q = smem + (c & 1) * kBuffer + kQ, *K = smem + (c & 1) * kBuffer + kK, *V = smem + (c & 1) * kBuffer + kV;
    if (tid == 0 && !p.state_only) {
      const uint32_t qa = smem_addr(Q), ka = smem_addr(K), sa = smem_addr(Ss);
#pragma unroll
      for (int part64 = 0; part64 < 2; ++part64)
        issue<2, 2>(tmem + kColA, operand(qa + part64 * kSub, 16), operand(ka + part64 * kSub, 16), instruction(128, false, false), 4,
                    part64);
#pragma unroll
      for (int part64 = 0; part64 < 2; ++part64)
        issue<2, 128>(tmem + kColB, operand(qa + part64 * kSub, 16), operand(sa + part64 * 4 * 2048, 16),
                      instruction(64, false, true), 4, part64);
      commit(bars);
    }
    next = c + 1 < chunks && starts(c + 1);
    if (c + 1 < chunks) load(c + 1);

    // episodes: the first token that this row's sums reach, and the state's
    unsigned m[4];
    bool flags = false;
#pragma unroll
    for (int w = 0; w < 4; ++w) m[w] = marks[w], flags |= m[w] != 0;
    int reach = 0, last = 0;
    bool carried = true;
    if (flags) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        // a start counts for its own token in token order, and behind it in reverse
        const unsigned before = w < part ? m[w] : w > part ? 0u : m[w] & ((lag ? 2u << lane : 1u << lane) - 1u);
        if (before) reach = 32 * w + 32 - lag - __clz(before), carried = false;
        if (m[w]) last = 32 * w + 32 - lag - __clz(m[w]);
      }
    }

    // the weighted V, half a token's row to a thread, in bf16 terms
    {
      const F2 w(token < rows && token >= last ? kept[rows - lag - token] : 0.f);
      const F2 less(-1.f);
      const bool third = s.parts > 2;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = 4 * half + k;
        const uint4 x = *block_of(V, token, j);
        const uint32_t in[4] = {x.x, x.y, x.z, x.w};
        uint32_t out[3][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          F2 y = mul(F2(__uint_as_float(in[e] << 16), __uint_as_float(in[e] & 0xffff0000u)), w);
#pragma unroll
          for (int term = 0; term < 3; ++term) {
            out[term][e] = pack(y.get().x, y.get().y);
            y = fma(F2(__uint_as_float(out[term][e] << 16), __uint_as_float(out[term][e] & 0xffff0000u)), less, y);
          }
        }
#pragma unroll
        for (int term = 0; term < 3; ++term)
          if (term < 2 || third)
            *block_of(W + term * kSub, token, j) = make_uint4(out[term][0], out[term][1], out[term][2], out[term][3]);
      }
    }
    fence_smem();
    __syncthreads();
    if (tid == 0) {
      const uint32_t wa = smem_addr(W), ka = smem_addr(K);
      issue<128, 128>(tmem + kColD, operand(ka, kSub), operand(wa, kSub), instruction(64 * s.parts, true, true), steps, false);
      commit(bars + 16);
    }

    F2 o[16], spoilt;
    if (!p.state_only) {
      lost |= !wait(bars, c & 1);
      fence_after();
      // P: the row's products with the keys, weighted, back to tensor memory; of
      // every 32 keys a thread takes 16.  All are on their way before the first is
      // used.
      float x[4][16];
#pragma unroll
      for (int k32 = 0; k32 < 4; ++k32)
        if (k32 <= part) load16(x[k32], mine + kColA + k32 * 32 + half * 16);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
      for (int k32 = 0; k32 < 4; ++k32) {
        const int key = k32 * 32 + half * 16;
        uint32_t y[8];
        if (k32 <= part) {
          float *z = x[k32];
#pragma unroll
          for (int j = 0; j < 16; ++j) asm volatile("" : "+f"(z[j]));
          if (k32 < part) {
            const F2 far(within[token - k32 * 32 - 31]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float4 f = ((const float4 *)fall)[half * 4 + j];
              const F2 u = mul(mul(F2(z[4 * j], z[4 * j + 1]), far), F2(f.x, f.y));
              const F2 v = mul(mul(F2(z[4 * j + 2], z[4 * j + 3]), far), F2(f.z, f.w));
              z[4 * j] = u.get().x, z[4 * j + 1] = u.get().y, z[4 * j + 2] = v.get().x, z[4 * j + 3] = v.get().y;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) z[j] *= within[token - key - j];
          }
          if (flags)
#pragma unroll
            for (int j = 0; j < 16; ++j) z[j] = key + j >= reach ? z[j] : 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = pack(z[2 * j], z[2 * j + 1]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = 0;
        }
        store8(mine + kColP + k32 * 16 + half * 8, y);
      }
      store_wait();
      fence_before();
      __syncthreads();
      fence_after();
      if (tid == 0) {
        const uint32_t va = smem_addr(V);
        issue_tmem<128>(tmem + kColC, tmem + kColP, operand(va, 16), instruction(64, false, true), steps);
        commit(bars + 8);
      }
      // B, weighted
      float z[32];
      load32(z, mine + kColB + 32 * half);
      load_wait<32>(z);
      const F2 w(flags && !carried ? 0.f : into[token + lag]);
#pragma unroll
      for (int j = 0; j < 16; ++j) o[j] = mul(F2(z[2 * j], z[2 * j + 1]), w);
    }

    // S
    const float left = rows == kRows ? whole.at(c) : expf(log_decay * rows);
    lost |= !wait(bars + 16, c & 1);
    fence_after();
    {
#pragma unroll
      for (int part16 = 0; part16 < 32; part16 += 16) {
        const uint32_t from = mine + kColD + col0 + part16;
        float x[16], y[16];
        load16(x, from);
        load16(y, from + 64);
        load_wait<16>(x);
        load_wait<16>(y);
        if (s.parts > 2) {  // the smallest terms first
          float z[16];
          load16(z, from + 128);
          load_wait<16>(z);
#pragma unroll
          for (int j = 0; j < 16; ++j) y[j] += z[j];
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) S[part16 + j] = (flags ? 0.f : S[part16 + j] * left) + (x[j] + y[j]);
      }
    }
    cut |= flags;
    if (flags)
#pragma unroll
      for (int j = 0; j < kN; j += 2) spoilt = fma(F2(S[j], S[j + 1]), F2(), spoilt);
    if (!p.state_only) {
      lost |= !wait(bars + 8, c & 1);
      fence_after();
      float x[32];
      load32(x, mine + kColC + 32 * half);
      load_wait<32>(x);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        o[j] = add(o[j], F2(x[2 * j], x[2 * j + 1]));
        spoilt = fma(o[j], F2(), spoilt);
      }
    }

    // Where a row or a state is not finite, it is summed again before S's copy in
    // shared memory is replaced.
    const bool here = token < rows && !p.state_only;
    const int64_t at_row = (((int64_t)b * p.time + origin + step * (c * kRows + token)) * p.heads + h) * s.vd + v0;
    bool mend = spoilt.sum() != 0.f;
    if (__syncthreads_or(mend)) {
      if (mend && here)
#pragma unroll 1
        for (int j = 32 * half; j < min(32 * half + 32, vd); ++j) {
          const float x = row_sum((const bf16 *)Q, (const bf16 *)K, (const bf16 *)V, (const bf16 *)Ss, token, j, reach,
                                  !flags || carried, kd, into[token + lag], within);
          if (s.out_float) ((float *)s.out)[at_row + j] = x;
          else ((bf16 *)s.out)[at_row + j] = from_float<bf16>(x);
        }
      if (mend && flags)
#pragma unroll 1
        for (int j = 0; j < kN; ++j) {
          const float x = state_sum((const bf16 *)K, (const bf16 *)V, last, rows, row, col0 + j, kept + rows - lag);
#pragma unroll
          for (int i = 0; i < kN; ++i) S[i] = i == j ? x : S[i];
        }
      __syncthreads();
    } else {
      mend = false;
    }
    if (c + 1 < chunks) {
      if (!p.state_only) publish();
      mark(next);
    }
    if (!p.state_only) {
      const unsigned skip = __ballot_sync(~0u, mend || !here);
      if (s.out_float) {
        if (!((skip >> lane) & 1))
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (32 * half + 4 * j < vd)
              *(float4 *)((float *)s.out + at_row + 32 * half + 4 * j) =
                  make_float4(o[2 * j].get().x, o[2 * j].get().y, o[2 * j + 1].get().x, o[2 * j + 1].get().y);
      } else {
        // through this thread's half row of W, which is free, then four lanes to a half row
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = pack(o[4 * j + e].get().x, o[4 * j + e].get().y);
          *block_of(W, token, 4 * half + j) = make_uint4(y[0], y[1], y[2], y[3]);
        }
        __syncwarp();
        const int r = lane / 4, block = 4 * half + lane % 4;
        const int64_t stride = (int64_t)step * p.heads * s.vd;
        bf16 *out = (bf16 *)s.out + at_row + (r - lane) * stride + block * 8;
#pragma unroll
        for (int i = 0; i < 32; i += 8, out += 8 * stride)
          if (!((skip >> (r + i)) & 1) && block * 8 < vd) *(uint4 *)out = *block_of(W, part * 32 + r + i, block);
      }
    }
  }

  asm volatile("cp.async.wait_all;" ::: "memory");
  fence_before();
  const bool stop = __syncthreads_or(lost);
  fence_after();
  if (stop && tid == 0) *status = call;
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*(const uint32_t *)(smem + kTmem)), "n"(kColumns));
  if (stop) return;

  if (p.state_only || (s.final && piece == p.pieces - 1)) {
    float *to = p.state_only ? p.states + p.states_at[which] + ((int64_t)bh * p.pieces + piece) * kd * s.vd
                             : s.final + (int64_t)bh * kd * s.vd;
    to += (int64_t)row * s.vd + v0 + col0;
    if (row < kd) {
#pragma unroll
      for (int j = 0; j < kN; j += 4)
        if (col0 + j < vd) *(float4 *)(to + j) = make_float4(S[j], S[j + 1], S[j + 2], S[j + 3]);
    }
  }
  if (p.state_only) {
    if (v0 == 0 && tid == 0)
      p.factors[((int64_t)which * p.batch * p.heads + bh) * p.pieces + piece] = cut ? 0.f : own ? Decay(log_decay * own).at(piece) : 1.f;
    return;
  }
  const int end = min(p.piece, p.time - s0);
  for (int r = own + warp; r < end; r += kThreads / 32) {
    const int64_t at = (((int64_t)b * p.time + s0 + r) * p.heads + h) * s.vd + v0;
    for (int col = lane; col < vd; col += 32) {
      if (s.out_float) ((float *)s.out)[at + col] = 0.f;
      else ((bf16 *)s.out)[at + col] = from_float<bf16>(0.f);
    }
  }
}
}  // namespace tc

int scan_tc_launch(const ScanParams &p, int *status, int call, cudaStream_t stream) {
  const cudaError_t rc = cudaFuncSetAttribute(tc::scan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, tc::kBytes);
  if (rc != cudaSuccess) return (int)rc;
  const int64_t grid = (int64_t)p.batch * p.heads * p.pieces * p.units;
  if (grid >= 1ll << 31) return (int)cudaErrorInvalidValue;
  tc::scan_kernel<<<(unsigned)grid, tc::kThreads, tc::kBytes, stream>>>(p, status, call);
  return (int)cudaGetLastError();
}

}  // namespace b200policy
