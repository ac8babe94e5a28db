// Decay attention: S_t = lambda S_{t-1} + k_t v_t^T, o_t = scale q_t S_t.  The
// one-token kernel, and the plans of the trajectory form (attention_scan.cuh).
//
// Backward, with R_t the cotangent of S_t:
//   R_t = scale q_t do_t^T + lambda [no episode starts at t+1] R_{t+1}
//   dq_t = scale S_t do_t,  dk_t = R_t v_t,  dv_t = R_t^T k_t
// Each is the forward pass's own scan with other tensors in its places: dq
// reads do, v, k (and S transposed); dk reads v, do, q and dv reads k, q, do,
// both with the tokens in reverse (heads of up to 64 in 16 bits take both from one
// walk).  One kernel runs all of them in one launch.
#include <algorithm>
#include <atomic>
#include "attention_scan.h"
#include "common.cuh"

namespace {
using namespace b200policy;

// ---- one token -----------------------------------------------------------------
// Bound by the state: [dk, dv] floats are read and written once, for 3 operations
// each.  A CTA takes one world and head.  A thread holds V columns (16 bytes where
// dv allows) of every kStepThreads / (dv / V)-th row, kBatch rows at a time in
// registers, so that a CTA has up to 16 KB of loads in flight and eight or more
// CTAs fit an SM; the rows' shares of q S meet in shared memory, in a fixed order.
// 16384 worlds, 4 heads of 64: 316 us, 6.9 TB/s; 1184 worlds, 6 heads of 48 and 96:
// 46 us, 5.8 TB/s.
constexpr int kStepThreads = 128, kBatch = 8;

template <class T, int V> __global__ void __launch_bounds__(kStepThreads) step_kernel(B200AttentionArgs a) {
  __shared__ float q[B200_HEAD_MAX], k[B200_HEAD_MAX];
  __shared__ float share[kStepThreads * V];
  struct alignas(4 * V) Block { float x[V]; };
  const int tid = threadIdx.x, b = blockIdx.x / a.heads, h = blockIdx.x % a.heads, hk = h / (a.heads / a.kv_heads);
  const int dk = a.dk, dv = a.dv, blocks = dv / V, rows = kStepThreads / blocks;  // rows at once
  const int r0 = tid / blocks, col = tid % blocks * V;
  const bool on = r0 < rows;
  const bool live = !a.lengths || a.lengths[b] > 0;
  const bool cut = live && a.first && a.first[b * a.first_batch];
  const int64_t plane = (int64_t)blockIdx.x * dk * dv;
  const float *from = a.state ? a.state + plane + col : nullptr;
  float *to = a.state_out + plane + col;
  Block s[kBatch];
  auto load = [&](int i0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int r = r0 + (i0 + i) * rows;
      if (on && r < dk && from && !cut) s[i] = *(const Block *)(from + r * dv);
      else
#pragma unroll
        for (int e = 0; e < V; ++e) s[i].x[e] = 0.f;
    }
  };
  load(0);
  if (tid < dk) {
    q[tid] = to_float(((const T *)a.q)[b * a.q_batch + h * a.q_head + tid]);
    k[tid] = to_float(((const T *)a.k)[b * a.k_batch + hk * a.k_head + tid]);
  }
  float v[V], o[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    v[e] = to_float(((const T *)a.v)[b * a.v_batch + hk * a.v_head + col + e]);
    o[e] = 0.f;
  }
  // above 1/2, lambda s = s + (lambda - 1) s: lambda itself, rounded, would be off by up
  // to 2^-25 for a slow decay, and a memory of n tokens by n times that; below, it is
  // lambda - 1 that loses what is left of s
  const float lambda = expf(a.log_decay[h]);
  const bool slow = lambda > 0.5f;
  const float factor = slow ? expm1f(a.log_decay[h]) : lambda;
  __syncthreads();
  for (int i0 = 0; i0 * rows < dk; i0 += kBatch) {
    if (i0) load(i0);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int r = r0 + (i0 + i) * rows;
      if (!on || r >= dk) continue;
      if (live)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          s[i].x[e] = fmaf(s[i].x[e], factor, slow ? s[i].x[e] : 0.f) + k[r] * v[e];
          o[e] += q[r] * s[i].x[e];
        }
      *(Block *)(to + r * dv) = s[i];
    }
  }
  if (on)
#pragma unroll
    for (int e = 0; e < V; ++e) share[r0 * dv + col + e] = o[e];
  __syncthreads();
  if (tid < dv) {
    float x = 0.f;
    for (int r = 0; r < rows; ++r) x += share[r * dv + tid];
    ((T *)a.out)[((int64_t)b * a.heads + h) * dv + tid] = from_float<T>(live ? x * a.scale : 0.f);
  }
}

// A long row's pieces: from the pieces' own states to the state before each
// piece, in place, and element by element.  A piece with an episode's start
// leaves nothing of what was before it (factor 0: selected, not multiplied).
__global__ void __launch_bounds__(128) pieces_kernel(const __grid_constant__ ScanParams p) {
  const Scan &s = p.scan[blockIdx.z];
  const int size = s.kd * s.vd, e = blockIdx.x * 128 + threadIdx.x;
  const int64_t bh = blockIdx.y;
  if (e >= size) return;
  const float *factor = p.factors + ((int64_t)blockIdx.z * gridDim.y + bh) * p.pieces;
  float carry = s.init ? s.init[bh * size + e / s.vd * s.init_row + e % s.vd * s.init_col] : 0.f;
  float *state = p.states + p.states_at[blockIdx.z] + bh * p.pieces * size + e;
  for (int i0 = 0; i0 < p.pieces; i0 += 8) {
    float own[8], f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      own[i] = i0 + i < p.pieces ? state[(int64_t)(i0 + i) * size] : 0.f;
      f[i] = i0 + i < p.pieces ? factor[i0 + i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i0 + i < p.pieces) state[(int64_t)(i0 + i) * size] = carry;
      carry = f[i] == 0.f ? own[i] : fmaf(f[i], carry, own[i]);
    }
  }
}

// dk and dv as sums over the query heads that share a key / value head, in head
// order: a warp to a token and head.
template <class T>
__global__ void __launch_bounds__(256) share_kernel(const float *part_k, const float *part_v, T *to_k, T *to_v, int64_t rows,
                                                    int group, int dk, int dv) {
  const int lane = threadIdx.x & 31;
  for (int64_t row = blockIdx.x * 8ll + (threadIdx.x >> 5); row < rows; row += gridDim.x * 8ll) {
    auto sum = [&](const float *part, T *to, int d) {
      part += row * group * d;
      to += row * d;
      for (int c = lane; c < d; c += 32) {
        float s = 0.f;
#pragma unroll 4
        for (int i = 0; i < group; ++i) s += part[i * d + c];
        to[c] = from_float<T>(s);
      }
    };
    sum(part_k, to_k, dk);
    sum(part_v, to_v, dv);
  }
}

constexpr int kSms = 148;
constexpr int kMostTokens = 0x7fffffff - 1024;  // of a row: token numbers a few chunks on are 32-bit too

bool aligned(const void *p, int64_t batch, int64_t time, int64_t head, int width, size_t bytes) {
  const int64_t block = 16 / (int64_t)bytes;
  return (uintptr_t)p % 16 == 0 && batch % block == 0 && time % block == 0 && head % block == 0 && width % block == 0;
}

struct Plan {
  ScanParams p;
  int kt, vt;
  bool tc;  // on tcgen05
  size_t float_rows;   // bytes of unreduced dk and dv
  size_t state_floats; // of p.states
  size_t bytes() const {
    return float_rows + (p.pieces > 1 ? (state_floats + (size_t)p.scans * p.batch * p.heads * p.pieces) * 4 : 0);
  }
};

void set_tensor(const void **p, int64_t *b, int64_t *t, int64_t *h, int *shared, int *vec, const void *x, int64_t sb,
                int64_t st, int64_t sh, int at_kv, int width, size_t bytes) {
  *p = x, *b = sb, *t = st, *h = sh, *shared = at_kv;
  *vec = aligned(x, sb, st, sh, width, bytes);
}

// What a launch of `count` scans does, up to where its workspace lies.
Plan plan_of(const B200AttentionArgs *a, bool backward) {
  Plan r{};
  ScanParams &p = r.p;
  const size_t bytes = element_bytes(a->dtype);
  const int group = a->heads / a->kv_heads;
  enum { Q, K, V, G };
  auto scan = [&](int q, int k, int v, int reverse) -> Scan & {
    Scan &s = p.scan[p.scans++];
    auto set = [&](int which, const void **ptr, int64_t *sb, int64_t *st, int64_t *sh, int *shared, int *vec) {
      switch (which) {
        case Q: set_tensor(ptr, sb, st, sh, shared, vec, a->q, a->q_batch, a->q_time, a->q_head, 0, a->dk, bytes); break;
        case K: set_tensor(ptr, sb, st, sh, shared, vec, a->k, a->k_batch, a->k_time, a->k_head, 1, a->dk, bytes); break;
        case V: set_tensor(ptr, sb, st, sh, shared, vec, a->v, a->v_batch, a->v_time, a->v_head, 1, a->dv, bytes); break;
        default: set_tensor(ptr, sb, st, sh, shared, vec, a->dout, a->g_batch, a->g_time, a->g_head, 0, a->dv, bytes);
      }
    };
    set(q, &s.q, &s.q_batch, &s.q_time, &s.q_head, &s.q_shared, &s.vec_q);
    set(k, &s.k, &s.k_batch, &s.k_time, &s.k_head, &s.k_shared, &s.vec_k);
    set(v, &s.v, &s.v_batch, &s.v_time, &s.v_head, &s.v_shared, &s.vec_v);
    s.reverse = reverse;
    s.kd = k == K || k == Q ? a->dk : a->dv;
    s.vd = v == K || v == Q ? a->dk : a->dv;
    s.pair_scale = reverse ? a->scale : 1.f;
    s.out_scale = reverse ? 1.f : a->scale;
    return s;
  };
  auto out = [&](Scan &s, void *to, bool wide) {
    s.out = to, s.out_float = wide;
    s.vec_out = (uintptr_t)to % 16 == 0 && s.vd % (wide || bytes == 4 ? 2 : 8) == 0;
  };
  if (!backward) {
    Scan &s = scan(Q, K, V, 0);
    s.init = a->state, s.init_row = a->dv, s.init_col = 1;
    s.final = a->state_out;
    out(s, a->out, false);
  } else {
    const size_t tokens = (size_t)a->batch * a->time * a->heads;
    float *wide = (float *)a->workspace;
    if (group > 1) r.float_rows = (tokens * (a->dk + a->dv) * 4 + 15) / 16 * 16;
    Scan &dq = scan(G, V, K, 0);  // dq_i = scale * sum w_ij (do_i . v_j) k_j + S do_i, and S transposed
    dq.init = a->state, dq.init_row = 1, dq.init_col = a->dv;
    out(dq, a->dq, false);
    // dk and dv walk the same state, dk its transpose: together where it fits
    const bool twin = bytes == 2 && a->dk <= 64 && a->dv <= 64;
    if (!twin) {
      Scan &dk = scan(V, G, Q, 1);
      dk.init = a->dstate_out, dk.init_row = 1, dk.init_col = a->dv;
      out(dk, group > 1 ? (void *)wide : a->dk_out, group > 1);
    }
    Scan &dv = scan(K, Q, G, 1);
    dv.init = a->dstate_out, dv.init_row = a->dv, dv.init_col = 1;
    dv.final = a->dstate;
    out(dv, group > 1 ? (void *)(wide + tokens * a->dk) : a->dv_out, group > 1);
    if (twin) {
      set_tensor(&dv.x, &dv.x_batch, &dv.x_time, &dv.x_head, &dv.x_shared, &dv.vec_x, a->v, a->v_batch, a->v_time, a->v_head, 1,
                 a->dv, bytes);
      dv.twin_out = group > 1 ? (void *)wide : a->dk_out;
      dv.vec_twin = (uintptr_t)dv.twin_out % 16 == 0 && a->dk % (group > 1 ? 2 : 8) == 0;
    }
  }
  p.log_decay = a->log_decay;
  p.first = a->first, p.first_batch = a->first_batch, p.first_time = a->first_time;
  p.lengths = a->lengths;
  p.batch = a->batch, p.time = a->time, p.heads = a->heads, p.group = group;
  int widest = 0;
  for (int i = 0; i < p.scans; ++i) r.kt = std::max(r.kt, p.scan[i].kd), widest = std::max(widest, p.scan[i].vd);
  // Slices of v: 64 wide, or 32 where that is all there is; for wide heads also where
  // the last slice of 64 would be at most half full (300 rows of 200 tokens and 6 heads
  // in bf16: of 80 and 72, 936 us with gradients against 1010; 200 such rows of 96 and
  // 104, whose last slice is fuller, 782 against 720; forward with one slice, of 128 and
  // 64, 173 us in two against 146, of 128 and 48, 183 against 163), and for 32-bit ones,
  // whose states of 64 columns leave one CTA an SM (of 80 and 72, 746 us forward against
  // 1052; of 128, 1220 against 1256).
  const bool thin = r.kt > 64 && (a->dtype == B200_FP32 || (widest > 64 && widest <= 96));
  r.vt = widest <= 32 || thin ? 32 : 64;
  for (int i = 0; i < p.scans; ++i) {
    p.scan[i].vec_final = (uintptr_t)p.scan[i].final % 16 == 0;
    p.scan[i].slices = (p.scan[i].vd + r.vt - 1) / r.vt;
    p.units += p.scan[i].slices;
    p.scan[i].parts = p.scan[i].final ? 3 : 2;
  }
  // Long rows of wide bf16 heads: 16 rows of 2048 tokens and 4 heads of 128 train in
  // 299 us instead of 408, 32 of 1024 in 309 instead of 345; 128 of 256, of which
  // chunks of 128 leave two, would take 375 instead of 324.  Its waits are bounded:
  // without a status word, an expired one would pass unseen.
  r.tc = a->dtype == B200_BF16 && a->time >= 1024 && r.kt > 64 && a->status;
  for (int i = 0; i < p.scans; ++i) {
    const Scan &s = p.scan[i];
    r.tc = r.tc && s.vec_q && s.vec_k && s.vec_v && s.vec_out && s.vec_final && s.vd % 8 == 0;
  }
  if (r.tc) {
    r.vt = 64;
    p.units = 0;
    for (int i = 0; i < p.scans; ++i) p.units += p.scan[i].slices = (p.scan[i].vd + 63) / 64;
  }
  // Rows are split where they are fewer than the SMs, into as many pieces as are
  // resident at once, of two chunks at least.  A piece reads its keys and values
  // twice, about 1.4 times the work, and takes two launches more (256 rows of 256
  // tokens and 64 wide: 27 us whole, 93 in two pieces each).  From there on rows stay
  // whole however long they are: of 4000 tokens, 147 rows of 64 wide take 168 us in
  // pieces and 148 take 201; on tcgen05, with one CTA an SM, 74 rows of two slices take
  // 156 and 75 take 297, for a second wave of two CTAs.
  const int64_t rows = (int64_t)p.batch * p.heads * p.units;
  const int tile = r.tc ? kTcTile : kTile, chunks = (p.time + tile - 1) / tile;
  const int resident = r.tc ? 1
                            : by_dtype(a->dtype, [&](auto type) { return scan_resident<decltype(type)>(r.kt, r.vt); });
  int64_t pieces = rows && rows < kSms ? std::min<int64_t>((int64_t)resident * kSms / rows, chunks / 2) : 1;
  if (pieces < 2) pieces = 1;
  p.piece = pieces > 1 ? (int)((chunks + pieces - 1) / pieces) * tile : std::max(p.time, 1);
  p.pieces = pieces > 1 ? (int)(((int64_t)p.time + p.piece - 1) / p.piece) : 1;
  for (int i = 0; i < p.scans; ++i) {
    p.states_at[i] = (int64_t)r.state_floats;
    r.state_floats += (size_t)p.batch * p.heads * p.pieces * p.scan[i].kd * p.scan[i].vd;
  }
  if (p.pieces > 1) {
    p.states = (float *)((char *)a->workspace + r.float_rows);
    p.factors = p.states + r.state_floats;
  }
  return r;
}

std::atomic<unsigned> calls;

template <class T> int run(Plan &r, int *status, cudaStream_t stream) {
  const int call = (int)(++calls & 0x7fffffffu) | 1 << 30;  // not zero
  ScanParams &p = r.p;
  auto launch = [&] {
    if (r.tc) return scan_tc_launch(p, status, call, stream);
    const int last = p.scans - 1;
    if (!p.scan[last].twin_out) return scan_launch<T>(p, r.kt, r.vt, stream);
    // the scan with a twin output, the last, by itself; the ones before it together
    ScanParams one = p;
    one.scan[0] = p.scan[last], one.states_at[0] = p.states_at[last];
    if (p.factors) one.factors = p.factors + (int64_t)last * p.batch * p.heads * p.pieces;
    one.scans = 1, one.units = p.scan[last].slices;
    ScanParams rest = p;
    rest.scans = last, rest.units = p.units - one.units;
    const int rc = scan_launch<T>(rest, r.kt, r.vt, stream);
    return rc ? rc : scan_launch<T>(one, r.kt, r.vt, stream);
  };
  if (p.pieces > 1) {
    p.state_only = 1;
    int rc = launch();
    if (rc) return rc;
    int size = 0;
    for (int i = 0; i < p.scans; ++i) size = std::max(size, p.scan[i].kd * p.scan[i].vd);
    pieces_kernel<<<dim3((size + 127) / 128, p.batch * p.heads, p.scans), 128, 0, stream>>>(p);
    p.state_only = 0;
  }
  return launch();
}

bool args_ok(const B200AttentionArgs *a) {
  return a && dtype_ok(a->dtype) && a->batch >= 0 && a->time >= 0 && a->time <= kMostTokens && a->heads > 0 && a->kv_heads > 0 &&
         a->heads % a->kv_heads == 0 && a->dk > 0 && a->dv > 0 && a->dk <= B200_HEAD_MAX && a->dv <= B200_HEAD_MAX &&
         (int64_t)a->batch * a->heads < (1ll << 31);
}
// What a launch reads and writes is there (with elements to it: batch is not zero).
bool pointers_ok(const B200AttentionArgs *a, bool backward) {
  const bool tokens = !a->time || (a->q && a->k && a->v && (backward ? a->dout && a->dq && a->dk_out && a->dv_out : a->out != nullptr));
  return tokens && a->log_decay && (backward || a->state_out);
}
bool workspace_ok(const Plan &r, const void *workspace) { return !r.bytes() || (workspace && (uintptr_t)workspace % 16 == 0); }
}  // namespace

extern "C" {
size_t b200policy_attention_bytes(void) { return sizeof(B200AttentionArgs); }

size_t b200policy_attention_workspace(const B200AttentionArgs *a, int backward) {
  return args_ok(a) && a->batch ? plan_of(a, backward != 0).bytes() : 0;
}

int b200policy_attention_forward(const B200AttentionArgs *a, void *stream) {
  if (!args_ok(a)) return (int)cudaErrorInvalidValue;
  if (a->batch == 0) return 0;
  if (!pointers_ok(a, false)) return (int)cudaErrorInvalidValue;
  return by_dtype(a->dtype, [&](auto type) {
    using T = decltype(type);
    if (a->time != 1) {
      Plan r = plan_of(a, false);
      if (!workspace_ok(r, a->workspace)) return (int)cudaErrorInvalidValue;
      return run<T>(r, a->status, (cudaStream_t)stream);
    }
    const unsigned grid = (unsigned)(a->batch * a->heads);
    const bool blocks = a->dv % 4 == 0 && (uintptr_t)a->state % 16 == 0 && (uintptr_t)a->state_out % 16 == 0;
    if (blocks) step_kernel<T, 4><<<grid, kStepThreads, 0, (cudaStream_t)stream>>>(*a);
    else step_kernel<T, 1><<<grid, kStepThreads, 0, (cudaStream_t)stream>>>(*a);
    return (int)cudaGetLastError();
  });
}

int b200policy_attention_backward(const B200AttentionArgs *a, void *stream) {
  if (!args_ok(a)) return (int)cudaErrorInvalidValue;
  if (a->batch == 0) return 0;
  if (!pointers_ok(a, true)) return (int)cudaErrorInvalidValue;
  return by_dtype(a->dtype, [&](auto type) {
    using T = decltype(type);
    Plan r = plan_of(a, true);
    if (!workspace_ok(r, a->workspace)) return (int)cudaErrorInvalidValue;
    const int rc = run<T>(r, a->status, (cudaStream_t)stream);
    const int64_t tokens = (int64_t)a->batch * a->time;
    if (rc || !r.float_rows || !tokens) return rc;
    const int group = a->heads / a->kv_heads;
    const float *dk = (const float *)a->workspace, *dv = dk + tokens * a->heads * a->dk;
    const int64_t rows = tokens * a->kv_heads;
    share_kernel<<<(unsigned)std::min<int64_t>((rows + 7) / 8, kSms * 8), 256, 0, (cudaStream_t)stream>>>(
        dk, dv, (T *)a->dk_out, (T *)a->dv_out, rows, group, a->dk, a->dv);
    return (int)cudaGetLastError();
  });
}
}
