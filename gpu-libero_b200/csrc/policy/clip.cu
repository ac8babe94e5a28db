// Global gradient norm over many tensors, and clipping.
//   norm = sqrt(sum |g|^2),  dst = g * min(1, max_norm / (norm + eps))
//
// Memory bound: every gradient is read for the norm, read again once it is
// known, and written (340M bf16 values: 349 us, 91% of the copy bandwidth over the
// three).  The second pass walks backward, so that it begins with what the first
// one left in L2.  The tensors' table is a kernel argument (no
// copy to the device); they are cut into chunks that persistent CTAs take in
// turn, whatever the tensors' sizes.  Squares are summed in 64 bits (16 bytes'
// worth at a time in 32 bits where that is in range), in an order that the
// tensors' sizes fix; every CTA of the second pass adds the partial sums itself,
// which saves a launch between the passes.
#include <algorithm>
#include <memory>
#include <new>
#include "common.cuh"

namespace {
using namespace b200policy;

constexpr int kThreads = 256;
constexpr int kBlocks = 148 * 4;
constexpr int kBatch = 4;  // 16-byte loads of a thread in flight

template <int N> struct Table {
  const void *src[N];
  void *dst[N];
  int64_t count[N];
  int first[N + 1];  // chunk that a tensor starts with
  int8_t dtype[N];
  int tensors;
  int chunk;  // elements
};

// The tensor of a chunk.
template <int N> __device__ __forceinline__ int tensor_of(const Table<N> &table, int chunk) {
  int low = 0, high = table.tensors - 1;
  while (low < high) {
    const int mid = (low + high + 1) / 2;
    if (table.first[mid] <= chunk) low = mid;
    else high = mid - 1;
  }
  return low;
}

template <class F> __device__ __forceinline__ void by_type(int dtype, F f) {
  if (dtype == B200_FP32) f(float());
  else if (dtype == B200_FP16) f(__half());
  else f(__nv_bfloat16());
}

template <class T> struct alignas(16) Block {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

// Sum of the squares of 16 bytes of values.  fp16 squares lie between 2^-48 and
// 2^32.  Others are summed in 32 bits while the largest is between 2^-40 and
// 2^60: smaller ones beside it do not count.
template <class T> __device__ __forceinline__ double squares(const Block<T> &b) {
  float top = 0.f, s = 0.f;
#pragma unroll
  for (int e = 0; e < Block<T>::N; ++e) {
    const float x = to_float(b.v[e]);
    top = fmaxf(top, fabsf(x));
    s = fmaf(x, x, s);
  }
  if (std::is_same<T, __half>::value || top == 0.f || (top > 0x1p-40f && top < 0x1p60f)) return s;
  double d = 0.;
#pragma unroll
  for (int e = 0; e < Block<T>::N; ++e) {
    const double x = to_float(b.v[e]);
    d += x * x;
  }
  return d;
}

template <int N>
__global__ void __launch_bounds__(kThreads) squares_kernel(const __grid_constant__ Table<N> table, double *parts) {
  __shared__ double part[32];
  double s = 0.;
  for (int chunk = blockIdx.x; chunk < table.first[table.tensors]; chunk += gridDim.x) {
    const int n = tensor_of(table, chunk);
    const int64_t low = (int64_t)(chunk - table.first[n]) * table.chunk;
    const int size = (int)min((int64_t)table.chunk, table.count[n] - low);
    by_type(table.dtype[n], [&](auto type) {
      using T = decltype(type);
      const T *g = (const T *)table.src[n] + low;
      int done = 0;
      if ((uintptr_t)g % 16 == 0) {
        const int blocks = size / Block<T>::N;
        const Block<T> *from = (const Block<T> *)g;
        done = blocks * Block<T>::N;
        int i = threadIdx.x;
        for (; i + (kBatch - 1) * kThreads < blocks; i += kBatch * kThreads) {
          Block<T> b[kBatch];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) b[u] = from[i + u * kThreads];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) s += squares(b[u]);
        }
        for (; i < blocks; i += kThreads) s += squares(from[i]);
      }
#pragma unroll 4
      for (int i = done + threadIdx.x; i < size; i += kThreads) {
        const double x = to_float(g[i]);
        s += x * x;
      }
    });
  }
  s = block_sum(s, part);
  if (threadIdx.x == 0) parts[blockIdx.x] = s;
}

template <int N>
__global__ void __launch_bounds__(kThreads)
    scale_kernel(const __grid_constant__ Table<N> table, const double *parts, int count, float *norm, float max_norm,
                 float eps) {
  __shared__ double part[32];
  double s = 0.;
  for (int i = threadIdx.x; i < count; i += kThreads) s += parts[i];
  const float total = (float)sqrt(block_sum(s, part));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  const float f = max_norm / (total + eps);
  const float factor = f > 1.f ? 1.f : f;  // a norm that is not a number stays one
  for (int back = blockIdx.x; back < table.first[table.tensors]; back += gridDim.x) {
    const int chunk = table.first[table.tensors] - 1 - back, n = tensor_of(table, chunk);
    const int64_t low = (int64_t)(chunk - table.first[n]) * table.chunk;
    const int size = (int)min((int64_t)table.chunk, table.count[n] - low);
    by_type(table.dtype[n], [&](auto type) {
      using T = decltype(type);
      const T *g = (const T *)table.src[n] + low;
      T *to = (T *)table.dst[n] + low;
      int done = 0;
      if (((uintptr_t)g | (uintptr_t)to) % 16 == 0) {
        const int blocks = size / Block<T>::N;
        const Block<T> *from = (const Block<T> *)g;
        done = blocks * Block<T>::N;
        auto put = [&](Block<T> b, int i) {
#pragma unroll
          for (int e = 0; e < Block<T>::N; ++e) b.v[e] = from_float<T>(to_float(b.v[e]) * factor);
          ((Block<T> *)to)[i] = b;
        };
        int i = threadIdx.x;
        for (; i + (kBatch - 1) * kThreads < blocks; i += kBatch * kThreads) {
          Block<T> b[kBatch];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) b[u] = from[i + u * kThreads];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) put(b[u], i + u * kThreads);
        }
        for (; i < blocks; i += kThreads) put(from[i], i);
      }
#pragma unroll 4
      for (int i = done + threadIdx.x; i < size; i += kThreads) to[i] = from_float<T>(to_float(g[i]) * factor);
    });
  }
}

// Tensors of one launch: a small table for most models, and the largest that a
// kernel's arguments hold (32,764 bytes).
constexpr int kFew = 96, kMany = 1000;
static_assert(sizeof(Table<kMany>) < 32000, "kernel arguments");

// Whether memory that is written is also read or written through another entry (0 or
// 1), or an error: CTAs take the entries in no order, so such a value would be scaled
// once or twice by chance.
int shares_memory(const B200ClipTensor *t, int count) {
  struct Range {
    uintptr_t low, high;
    bool write;
  } few[2 * kFew];
  std::unique_ptr<Range[]> many(count > kFew ? new (std::nothrow) Range[2 * (size_t)count] : nullptr);
  Range *ranges = count > kFew ? many.get() : few;
  if (!ranges) return -(int)cudaErrorMemoryAllocation;
  size_t n = 0;
  for (int i = 0; i < count; ++i) {
    if (!t[i].count) continue;
    const size_t size = (size_t)t[i].count * element_bytes((int)t[i].dtype);
    ranges[n++] = {(uintptr_t)t[i].dst, (uintptr_t)t[i].dst + size, true};
    if (t[i].src != t[i].dst) ranges[n++] = {(uintptr_t)t[i].src, (uintptr_t)t[i].src + size, false};
  }
  std::sort(ranges, ranges + n, [](const Range &a, const Range &b) { return a.low < b.low; });
  uintptr_t written = 0, taken = 0;  // ends of what has been written, and of all
  for (size_t i = 0; i < n; ++i) {
    if (ranges[i].low < (ranges[i].write ? taken : written)) return 1;
    taken = std::max(taken, ranges[i].high);
    if (ranges[i].write) written = std::max(written, ranges[i].high);
  }
  return 0;
}

int per_launch(int count) { return count <= kFew ? kFew : kMany; }
int launches(int count) { return std::max(1, (count + per_launch(count) - 1) / per_launch(count)); }

// Chunks of 16,384 elements; smaller ones where that would leave CTAs idle.
template <int N> void fill(Table<N> &table, const B200ClipTensor *t, int count) {
  int64_t total = 0;
  for (int i = 0; i < count; ++i) total += t[i].count;
  table.chunk = 16384;
  while (table.chunk > 2048 && total / table.chunk < kBlocks) table.chunk /= 2;
  int64_t chunks = 0;
  do {  // (chunk numbers are 32-bit)
    chunks = 0;
    for (int i = 0; i < count; ++i) chunks += (t[i].count + table.chunk - 1) / table.chunk;
    if (chunks > 1 << 30) table.chunk *= 2;
  } while (chunks > 1 << 30);
  table.tensors = count;
  table.first[0] = 0;
  for (int i = 0; i < count; ++i) {
    table.src[i] = t[i].src, table.dst[i] = t[i].dst, table.count[i] = t[i].count;
    table.dtype[i] = (int8_t)t[i].dtype;
    table.first[i + 1] = table.first[i] + (int)((t[i].count + table.chunk - 1) / table.chunk);
  }
}

template <int N>
int run(const B200ClipTensor *tensors, int count, float max_norm, float eps, float *norm, double *parts, cudaStream_t s) {
  Table<N> table;
  const int many = launches(count);
  auto take = [&](int l) { fill(table, tensors + l * N, std::min(N, count - l * N)); };
  auto blocks = [&] { return std::max(1, std::min(kBlocks, table.first[table.tensors])); };
  int sums = 0;
  for (int l = 0; l < many; ++l) {
    take(l);
    squares_kernel<N><<<blocks(), kThreads, 0, s>>>(table, parts + sums);
    sums += blocks();
  }
  for (int l = many - 1; l >= 0; --l) {
    if (l < many - 1) take(l);
    scale_kernel<N><<<blocks(), kThreads, 0, s>>>(table, parts, sums, l == 0 ? norm : nullptr, max_norm, eps);
  }
  return (int)cudaGetLastError();
}
}  // namespace

extern "C" {
size_t b200policy_clip_bytes(void) { return sizeof(B200ClipTensor); }

size_t b200policy_clip_workspace(const B200ClipTensor *, int count) {
  return count < 0 ? 0 : (size_t)launches(count) * kBlocks * sizeof(double);
}

int b200policy_clip(const B200ClipTensor *tensors, int count, float max_norm, float eps, float *norm, void *workspace,
                    void *stream) {
  if (count < 0 || (count && !tensors) || !norm || !workspace) return (int)cudaErrorInvalidValue;
  for (int i = 0; i < count; ++i)
    if (tensors[i].count < 0 || tensors[i].dtype < B200_FP32 || tensors[i].dtype > B200_BF16 ||
        (tensors[i].count && !(tensors[i].src && tensors[i].dst)))
      return (int)cudaErrorInvalidValue;
  if (const int shared = shares_memory(tensors, count)) return shared < 0 ? -shared : (int)cudaErrorInvalidValue;
  return per_launch(count) == kFew ? run<kFew>(tensors, count, max_norm, eps, norm, (double *)workspace, (cudaStream_t)stream)
                                   : run<kMany>(tensors, count, max_norm, eps, norm, (double *)workspace, (cudaStream_t)stream);
}

const char *b200policy_source_id(void) { return B200POLICY_SOURCE_ID; }
int b200policy_arch(void) { return 100; }
}
