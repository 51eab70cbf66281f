// Dropout whose mask is a function of (key, site, element index) and is never stored: the backward pass computes it
// again.  Optionally with the residual sum that follows it in a block:  y = residual + keep x / (1 - q).
//
// Generator: Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3",
// 2011).  Counter (i low, i high, site, 0) with i = element index / 8 and the 64-bit key read from device memory (a
// captured graph can be replayed under a new key) gives four words = eight 16-bit draws; element 8 i + 2 j takes the low
// half of word j, element 8 i + 2 j + 1 the high half.  An element is dropped iff its draw is below q 65536, q = p
// rounded to a multiple of 2^-16, and the kept ones are scaled by 1 / (1 - q): the expectation is exact.
//
// Bound by memory: one 32-bit word per element would make it issue-bound (128 Mi bf16 elements, 2 x 256 MB: 113 us
// against 84.1 us with 16-bit draws and 83.8 us for the same loop without a generator).  Four independent 16-byte
// runs per thread and iteration keep enough loads in flight.  16384 x 4096 bf16 with a residual 68.5 us, its gradient 47.6.  Where one of
// the tensors does not start on a 16-byte boundary all are taken element by element (64 Mi bf16 132 us against 47, fp32 202 against 84).
#include "block_calls.h"
#include "launch.cuh"
#include "vec.cuh"

#define DROP_THREADS 256
#define DROP_RUNS 4      // runs of eight elements per thread and iteration

__device__ __forceinline__ uint4 philox4x32_10(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// bit e of the result: element e of the run is kept
__device__ __forceinline__ uint32_t drop_keep_bits(long long run, uint32_t site, uint32_t k0, uint32_t k1, uint32_t drop) {
  const uint4 w = philox4x32_10((uint32_t)run, (uint32_t)(run >> 32), site, 0u, k0, k1);
  const uint32_t q[4] = {w.x, w.y, w.z, w.w};
  uint32_t bits = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    bits |= (uint32_t)((q[j] & 0xFFFFu) >= drop) << (2 * j);
    bits |= (uint32_t)((q[j] >> 16) >= drop) << (2 * j + 1);
  }
  return bits;
}

// eight consecutive elements, A of them per access
template <typename T, int A>
__device__ __forceinline__ void run_load(const T* p, Vec<T, A> (&v)[8 / A]) {
#pragma unroll
  for (int j = 0; j < 8 / A; ++j) v[j].load(p + j * A);
}

template <typename T, int A, bool RES>
__global__ void __launch_bounds__(DROP_THREADS) dropout_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                               T* __restrict__ y, long long n, const uint32_t* key,
                                                               uint32_t site, uint32_t drop, float scale) {
  pdl_wait();
  pdl_trigger();
  const uint32_t k0 = key[0], k1 = key[1];
  const long long runs = n / 8, step = (long long)gridDim.x * DROP_THREADS * DROP_RUNS;
  for (long long r0 = (long long)blockIdx.x * DROP_THREADS * DROP_RUNS + threadIdx.x; r0 < runs; r0 += step) {
    Vec<T, A> v[DROP_RUNS][8 / A], w[DROP_RUNS][8 / A];
#pragma unroll
    for (int u = 0; u < DROP_RUNS; ++u) {
      const long long r = r0 + u * DROP_THREADS;
      if (r < runs) {
        run_load<T, A>(x + r * 8, v[u]);
        if (RES) run_load<T, A>(res + r * 8, w[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < DROP_RUNS; ++u) {
      const long long r = r0 + u * DROP_THREADS;
      if (r < runs) {
        const uint32_t keep = drop_keep_bits(r, site, k0, k1, drop);
#pragma unroll
        for (int j = 0; j < 8 / A; ++j) {
          Vec<T, A> o;
#pragma unroll
          for (int e = 0; e < A; ++e) {
            const bool k = (keep >> (j * A + e)) & 1u;
            const float f = to_f(v[u][j].e[e]);
            if (RES) o.e[e] = k ? from_f<T>(fmaf(f, scale, to_f(w[u][j].e[e]))) : w[u][j].e[e];
            else o.e[e] = from_f<T>(k ? f * scale : 0.f);
          }
          o.store(y + r * 8 + j * A);
        }
      }
    }
  }
  // the last n % 8 elements
  if (blockIdx.x == 0 && threadIdx.x == 0 && runs * 8 < n) {
    const uint32_t keep = drop_keep_bits(runs, site, k0, k1, drop);
    for (int e = 0; runs * 8 + e < n; ++e) {
      const long long i = runs * 8 + e;
      const bool k = (keep >> e) & 1u;
      const float f = to_f(x[i]);
      if (RES) y[i] = k ? from_f<T>(fmaf(f, scale, to_f(res[i]))) : res[i];
      else y[i] = from_f<T>(k ? f * scale : 0.f);
    }
  }
}

template <typename T>
static int dropout_launch(const void* x, const void* res, void* y, long long n, const void* key, uint32_t site,
                          uint32_t drop, float scale, cudaStream_t st) {
  const uintptr_t bits = (uintptr_t)x | (uintptr_t)res | (uintptr_t)y;
  constexpr int W = 16 / sizeof(T);
  long long blocks = (n / 8 + DROP_THREADS * DROP_RUNS - 1) / (DROP_THREADS * DROP_RUNS);
  // 32 blocks per SM in all, four generations of the eight that are resident
  if (blocks > 32LL * sm_count()) blocks = 32LL * sm_count();
  if (blocks < 1) blocks = 1;
  const T *px = reinterpret_cast<const T*>(x), *pr = reinterpret_cast<const T*>(res);
  T* py = reinterpret_cast<T*>(y);
  const uint32_t* k = reinterpret_cast<const uint32_t*>(key);
  const dim3 g((unsigned)blocks), b(DROP_THREADS);
  if (bits % 16 == 0) {
    return (int)(res != nullptr ? launch_k(dropout_kernel<T, W, true>, g, b, 0, st, px, pr, py, n, k, site, drop, scale)
                                : launch_k(dropout_kernel<T, W, false>, g, b, 0, st, px, pr, py, n, k, site, drop, scale));
  }
  return (int)(res != nullptr ? launch_k(dropout_kernel<T, 1, true>, g, b, 0, st, px, pr, py, n, k, site, drop, scale)
                              : launch_k(dropout_kernel<T, 1, false>, g, b, 0, st, px, pr, py, n, k, site, drop, scale));
}

extern "C" int dropout_apply(DropoutCall* c) {
  if (c->n <= 0 || c->drop < 0 || c->drop > 65536 || ((uintptr_t)c->key & 3) != 0) return -1;
  c->launches = 1;
  const float scale = c->drop < 65536 ? 65536.f / (65536.f - (float)c->drop) : 0.f;      // 65536: no draw reaches it, nothing is kept
  const uint32_t site = (uint32_t)c->site, drop = (uint32_t)c->drop;
  if (c->dt == DT_F32) return dropout_launch<float>(c->x, c->res, c->y, c->n, c->key, site, drop, scale, (cudaStream_t)c->stream);
  if (c->dt == DT_BF16) return dropout_launch<__nv_bfloat16>(c->x, c->res, c->y, c->n, c->key, site, drop, scale, (cudaStream_t)c->stream);
  if (c->dt == DT_F16) return dropout_launch<__half>(c->x, c->res, c->y, c->n, c->key, site, drop, scale, (cudaStream_t)c->stream);
  return -1;
}
