// Layer normalisation over the last dimension (width D) of an [N, D] matrix, forward and backward.
//
//   mu = mean(x), var = mean((x - mu)^2), rs = 1 / sqrt(var + eps), z = (x - mu) rs, y = z w + b
//   g = dy w;  dx = rs (g - mean(g) - z mean(g z));  dw = sum over rows of dy z;  db = sum over rows of dy
//
// Both directions are one pass over memory: a row is read once, kept on the SM (the variance is taken about the mean, not from
// a sum of squares, and z from x - mu, not from x rs - mu rs: 1 % of the time at 16384 x 4096 bf16) and written once.  All statistics
// and sums are fp32.
//
// Forward: a row belongs to one warp (up to 64 bytes x 16 per lane as they lie in memory, no block barrier), to several for long
// rows and where there are few rows; blocks walk over the rows with weight and bias in shared memory.
//
// Backward: a row belongs to a group of 32 .. 1024 threads, so that a thread's share of the columns is small enough to keep
// the running sums of dw and db of all its rows in registers.  Rows that start on 16-byte boundaries come through a ring of
// bulk copies in shared memory (three rows of x and dy per group under way); others are read into registers.  A block adds its
// groups in shared memory and writes one partial row; a second kernel adds the partial rows in block order.  No atomics: the same
// inputs give the same bits.
//
// Bound by memory for fp32: 16384 x 2048 forward 48 us (268 MB, 0.87 of the copy rate), backward with its reduction 67 (403 MB, 0.93).
// 16-bit rows by the latency of a row's steps (load, sum, squares, scaling, with a barrier between them) at 24 warps per SM: 16384 x 4096
// bf16 forward 53 us (0.78), backward 88 (0.71), with 54 % of the issue slots and half of the memory's cycles in use.  Small ones by
// launch and latency: 1120 x 650 fp32 16 us for the three kernels.
//
// Rows that do not start on 16-byte boundaries take narrower accesses (V elements at a time; 65536 x 1027 fp16 17 and 25 % of the copy
// rate); of long rows, above 4096 elements forward (8192 where they are not off boundaries) and 8192 backward, a part of 0.1 to 0.9 KB per
// thread spills to local memory; rows too long for registers (above 16384 elements) take the *_long kernels, which read the row again from L2, one element per access (4096 x 20000 bf16,
// forward and backward 763 us, the library 418; 2048 x 20000 fp32 469 and 353).
#include "block_calls.h"
#include "launch.cuh"
#include "tc_common.cuh"
#include "vec.cuh"

#include <atomic>

#define LN_MAX_ROW 16384

// A wait of the rings is bounded.  A warp whose wait runs out sets the error word and goes on in ln_fwd_late or ln_bwd_late: it waits
// no more, meets its group's barriers with NaN for its share of the sums, so that the group's remaining rows become NaN as a whole, and its
// columns of dw and db are NaN.  The thread that starts the copies also waits for those in flight and starts none again.
__device__ int g_ln_error;

struct LnArgs {
  const void* x;        // [N, D], ldx elements per row
  const void* w;        // [D] or null (ones)
  const void* b;        // [D] or null (zeros)
  void* y;              // [N, D] contiguous
  float* mean;          // [N]
  float* rstd;          // [N]
  const void* dy;       // [N, D], lddy elements per row
  void* dx;             // [N, D] contiguous, or null
  float* partial;       // [blocks][2][D], or null
  long long n, ldx, lddy;
  int d, w_dt;
  float eps;
};

__device__ __forceinline__ float ln_warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// barrier of one row group (a whole number of warps); a one-warp group needs no block barrier
__device__ __forceinline__ void ln_group_sync(int group, int threads) {
  if (threads == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory");
}
// sums of NS values over a row group, fixed order; red: [2][NS][warps per group], buffers used in turn by successive calls
template <int NS>
__device__ __forceinline__ void ln_group_sum(float (&v)[NS], float* red, int group, int t, int threads) {
#pragma unroll
  for (int k = 0; k < NS; ++k) v[k] = ln_warp_sum(v[k]);
  const int warps = threads >> 5;
  if (warps == 1) return;
  if ((t & 31) == 0) {
#pragma unroll
    for (int k = 0; k < NS; ++k) red[k * 32 + (t >> 5)] = v[k];
  }
  ln_group_sync(group, threads);
#pragma unroll
  for (int k = 0; k < NS; ++k) v[k] = ln_warp_sum((t & 31) < warps ? red[k * 32 + (t & 31)] : 0.f);
}

// column of element e of thread t: vectors of V elements, T threads side by side
template <int V>
__device__ __forceinline__ int ln_col(int t, int threads, int e) { return ((e / V) * threads + t) * V + (e % V); }

template <typename T, int V, int E>
__device__ __forceinline__ void ln_load(const T* row, int d, int t, int threads, float (&out)[E]) {
#pragma unroll
  for (int j = 0; j < E / V; ++j) {
    const int c = (j * threads + t) * V;
    Vec<T, V> v;
    v.clear();
    if (c < d) v.load(row + c);
#pragma unroll
    for (int k = 0; k < V; ++k) out[j * V + k] = to_f(v.e[k]);
  }
}

// value `c` of a parameter (`none` without it)
__device__ __forceinline__ float ln_param(const void* p, int dt, int c, float none) {
  return p != nullptr ? load_any(p, dt, c) : none;
}
// parameters wait in shared memory as fp32 in four-element pieces: piece h of vector v at (h vectors + v), so that consecutive
// lanes read consecutive 16-byte units
template <int V>
__device__ __forceinline__ void ln_get(const float* s, int vectors, int v, float (&out)[V]) {
  if (V >= 4) {
#pragma unroll
    for (int h = 0; h < V / 4; ++h) {
      const float4 q = reinterpret_cast<const float4*>(s)[h * vectors + v];
      out[(4 * h) % V] = q.x; out[(4 * h + 1) % V] = q.y; out[(4 * h + 2) % V] = q.z; out[(4 * h + 3) % V] = q.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) out[k] = s[v * V + k];
  }
}
template <int V>
__device__ __forceinline__ int ln_slot(int vectors, int c) {      // where element c is kept
  return V >= 4 ? ((c % V / 4) * vectors + c / V) * 4 + c % 4 : c;
}

#define LN_RING 3        // rows of a group under way (backward)
#define LN_T16 640       // threads of a block with 16 elements per thread (96 registers)

__device__ __forceinline__ void ln_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
#define LN_NAN __int_as_float(0x7FC00000)
// where a group stands: its row, the stage k of that row and the parity of its barrier; depth stages, copies of `ahead` rows under way
struct LnRing {
  uint64_t* full;
  int k, depth, ahead;
  uint32_t phase;
  long long row, stride, n;
};
__device__ __forceinline__ void ln_gave_up(const LnRing& r, int t) {
  atomicExch(&g_ln_error, 1);
  if (t != 0) return;
  for (int j = 0; j < r.ahead && r.row + j * r.stride < r.n; ++j)
    mbar_wait(r.full + (r.k + j) % r.depth, r.phase ^ (r.k + j >= r.depth ? 1u : 0u));
}
template <typename T>
__device__ __forceinline__ void ln_nan_row(T* row, int d, int t, int threads) {
  constexpr int V = 16 / sizeof(T);
  for (int v = t; v < d / V; v += threads)
    for (int e = 0; e < V; ++e) row[v * V + e] = from_f<T>(LN_NAN);
}
template <typename T>
__device__ __noinline__ void ln_fwd_late(LnRing r, float* red, T* y, float* mean, float* rstd, int d, int group, int t, int threads) {
  ln_gave_up(r, t);
  for (long long row = r.row; row < r.n; row += r.stride) {
    float s[1] = {LN_NAN};
    ln_group_sum<1>(s, red, group, t, threads);
    ln_group_sum<1>(s, red + 32, group, t, threads);
    ln_nan_row(y + row * d, d, t, threads);
    if (t == 0 && mean != nullptr) mean[row] = rstd[row] = LN_NAN;
  }
}
template <typename T>
__device__ __noinline__ void ln_bwd_late(LnRing r, int turn, float* red, T* dx, int d, int group, int t, int threads) {
  ln_gave_up(r, t);
  for (long long row = r.row; row < r.n; row += r.stride, turn ^= 1) {
    float s[2] = {LN_NAN, LN_NAN};
    ln_group_sum<2>(s, red + turn * 64, group, t, threads);
    if (dx != nullptr) ln_nan_row(dx + row * d, d, t, threads);
  }
}

// parameters of vector v as pairs
template <int V>
__device__ __forceinline__ void ln_get2(const float* s, int vectors, int v, F2 (&out)[V / 2]) {
#pragma unroll
  for (int h = 0; h < V / 4; ++h) {
    const float4 q = reinterpret_cast<const float4*>(s)[h * vectors + v];
    out[2 * h] = f2(q.x, q.y);
    out[2 * h + 1] = f2(q.z, q.w);
  }
}

// Rows on 16-byte boundaries, four vectors per lane.  A group (one warp up to 1024 16-bit elements) has two rows or more of its
// own coming into shared memory by bulk copies while it works on a third in registers; the stage is filled again as soon as
// the registers have it.  Arithmetic in pairs of fp32 numbers, which halves the instructions (16384 x 4096 bf16: one element at a time 85
// us, with pairs and 8 vectors per lane 77, with 4 vectors 63, with 768 threads 57, with one vote per row on the wait 53; 65536 x 1024: 46).
// GIVE_UP: the first wait counts as one that ran out (tests).
template <typename T, int NV, bool GIVE_UP>
__global__ void __launch_bounds__(768, 1) ln_fwd_ring_kernel(LnArgs a, int threads, int groups, int depth) {
  constexpr int V = 16 / sizeof(T);
  extern __shared__ float4 ln_smem4[];
  __shared__ float red[24][2][32];
  __shared__ uint64_t full[24][8];
  const int vectors = a.d / V, row_bytes = vectors * 16;
  float *w_s = reinterpret_cast<float*>(ln_smem4), *b_s = w_s + a.d;
  const int group = threadIdx.x / threads, t = threadIdx.x % threads;
  uint8_t* mine = reinterpret_cast<uint8_t*>(b_s + a.d) + (long long)group * depth * row_bytes;
  if (t == 0) {
    for (int k = 0; k < depth; ++k) mbar_init(&full[group][k], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_trigger();
  const T* x = reinterpret_cast<const T*>(a.x);
  const long long first = (long long)blockIdx.x * groups + group, stride = (long long)gridDim.x * groups;
  const auto fill = [&](long long row, int k) {
    mbar_expect_tx(&full[group][k], row_bytes);
    ln_bulk(mine + k * row_bytes, x + row * a.ldx, row_bytes, &full[group][k]);
  };
  if (t == 0)
    for (int k = 0; k < depth; ++k)
      if (first + k * stride < a.n) fill(first + k * stride, k);
  for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
    w_s[ln_slot<V>(vectors, c)] = ln_param(a.w, a.w_dt, c, 1.f);
    b_s[ln_slot<V>(vectors, c)] = ln_param(a.b, a.w_dt, c, 0.f);
  }
  __syncthreads();
  const float inv_d = 1.f / (float)a.d;
  int k = 0;
  uint32_t phase = 0;
  for (long long row = first; row < a.n; row += stride) {
    if (GIVE_UP || !__all_sync(0xffffffffu, mbar_wait(&full[group][k], phase))) {
      ln_fwd_late({full[group], k, depth, depth, phase, row, stride, a.n}, red[group][0], reinterpret_cast<T*>(a.y), a.mean, a.rstd, a.d,
                  group, t, threads);
      break;
    }
    Vec<T, V> r[NV];
    F2 sum = f2(0.f), more = f2(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      r[j].clear();
      if (j * threads + t < vectors) r[j].load(reinterpret_cast<const T*>(mine + k * row_bytes) + (j * threads + t) * V);
#pragma unroll
      for (int i = 0; i < V / 2; i += 2) {
        sum = sum + pair_of(r[j], i);
        more = more + pair_of(r[j], i + 1);
      }
    }
    float s[1] = {f2_sum(sum) + f2_sum(more)};
    ln_group_sum<1>(s, red[group][0], group, t, threads);      // every thread has the row in registers
    if (t == 0 && row + depth * stride < a.n) fill(row + depth * stride, k);
    const float mu = s[0] * inv_d;
    sum = more = f2(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) opaque(r[j].raw);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * threads + t < vectors) {
#pragma unroll
        for (int i = 0; i < V / 2; i += 2) {
          const F2 p = pair_of(r[j], i) + f2(-mu), q = pair_of(r[j], i + 1) + f2(-mu);
          sum = f2_fma(p, p, sum);
          more = f2_fma(q, q, more);
        }
      }
    s[0] = f2_sum(sum) + f2_sum(more);
    ln_group_sum<1>(s, red[group][1], group, t, threads);
    const float rs = 1.f / sqrtf(fmaf(s[0], inv_d, a.eps));
    const F2 rs2 = f2(rs), off = f2(-mu);
    T* y = reinterpret_cast<T*>(a.y) + row * a.d;
#pragma unroll
    for (int j = 0; j < NV; ++j) opaque(r[j].raw);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * threads + t < vectors) {
        F2 w[V / 2], b[V / 2];
        ln_get2<V>(w_s, vectors, j * threads + t, w);
        ln_get2<V>(b_s, vectors, j * threads + t, b);
        F2 o[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) o[i] = f2_fma((pair_of(r[j], i) + off) * rs2, w[i], b[i]);
        store_pairs(y + (j * threads + t) * V, o);
      }
    if (t == 0 && a.mean != nullptr) {
      a.mean[row] = mu;
      a.rstd[row] = rs;
    }
    if (++k == depth) { k = 0; phase ^= 1; }
  }
}

// Other rows, and few rows: up to 32 V NV elements per warp, in registers.
template <typename T, int V, int NV>
__global__ void __launch_bounds__(256, NV >= 16 ? 2 : 4) ln_fwd_kernel(LnArgs a, int threads, int groups) {
  extern __shared__ float4 ln_smem4[];
  float *w_s = reinterpret_cast<float*>(ln_smem4), *b_s = w_s + (a.d + V - 1) / V * V;
  __shared__ float red[8][2][32];   // [group][buffer][warp]
  const int group = threadIdx.x / threads, t = threadIdx.x % threads, vectors = (a.d + V - 1) / V;
  pdl_wait();
  pdl_trigger();
  const T* x = reinterpret_cast<const T*>(a.x);
  const float inv_d = 1.f / (float)a.d;
  const long long first = (long long)blockIdx.x * groups + group, stride = (long long)gridDim.x * groups;
  Vec<T, V> r[NV];
  const auto load = [&](long long row) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      r[j].clear();
      if (j * threads + t < vectors) r[j].load(x + row * a.ldx + (j * threads + t) * V);
    }
  };
  if (first < a.n) load(first);
  for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
    w_s[ln_slot<V>(vectors, c)] = ln_param(a.w, a.w_dt, c, 1.f);
    b_s[ln_slot<V>(vectors, c)] = ln_param(a.b, a.w_dt, c, 0.f);
  }
  __syncthreads();
  for (long long row = first; row < a.n; row += stride) {
    if (row != first) load(row);
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) s[0] += to_f(r[j].e[k]);
    ln_group_sum<1>(s, red[group][0], group, t, threads);
    const float mu = s[0] * inv_d;
    s[0] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) opaque(r[j].raw);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * threads + t < vectors) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float v = to_f(r[j].e[k]) - mu;
          s[0] = fmaf(v, v, s[0]);
        }
      }
    ln_group_sum<1>(s, red[group][1], group, t, threads);
    const float rs = 1.f / sqrtf(fmaf(s[0], inv_d, a.eps));
    T* y = reinterpret_cast<T*>(a.y) + row * a.d;
#pragma unroll
    for (int j = 0; j < NV; ++j) opaque(r[j].raw);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * threads + t < vectors) {
        float w[V], b[V];
        ln_get<V>(w_s, vectors, j * threads + t, w);
        ln_get<V>(b_s, vectors, j * threads + t, b);
        Vec<T, V> o;
#pragma unroll
        for (int k = 0; k < V; ++k) o.e[k] = from_f<T>(fmaf((to_f(r[j].e[k]) - mu) * rs, w[k], b[k]));
        o.store(y + (j * threads + t) * V);
      }
    if (t == 0 && a.mean != nullptr) {
      a.mean[row] = mu;
      a.rstd[row] = rs;
    }
  }
}

// Rows on 16-byte boundaries.  x and dy of a row lie in a stage of the group's ring and are read there twice, before and after
// the row's two sums are known; registers hold only the sums of dw and db.  The stage
// of the row before is filled again behind the barrier of the row's sums: by then every thread is done with it.
template <typename T, int E, bool GIVE_UP>
__global__ void __launch_bounds__(E == 8 ? 1024 : LN_T16, 1) ln_bwd_ring_kernel(LnArgs a, int threads, int groups) {
  constexpr int V = 16 / sizeof(T), NV = E / V;
  extern __shared__ float4 ln_smem4[];
  __shared__ float red[16][2][64];
  __shared__ uint64_t full[16][LN_RING];
  const int vectors = a.d / V, row_bytes = vectors * 16;
  float* w_s = reinterpret_cast<float*>(ln_smem4);                       // [D], later [2][D] sums of the block's groups
  uint8_t* ring = reinterpret_cast<uint8_t*>(ln_smem4) + (a.d * 8 + 15) / 16 * 16;
  const int group = threadIdx.x / threads, t = threadIdx.x % threads;
  uint8_t* mine = ring + (long long)group * LN_RING * 2 * row_bytes;
  if (t == 0) {
    for (int k = 0; k < LN_RING; ++k) mbar_init(&full[group][k], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_trigger();
  const T *x = reinterpret_cast<const T*>(a.x), *dy = reinterpret_cast<const T*>(a.dy);
  for (int c = threadIdx.x; c < a.d; c += blockDim.x) w_s[ln_slot<V>(vectors, c)] = ln_param(a.w, a.w_dt, c, 1.f);
  __syncthreads();
  const long long first = (long long)blockIdx.x * groups + group, stride = (long long)gridDim.x * groups;
  const auto fill = [&](long long row, int k) {
    mbar_expect_tx(&full[group][k], 2 * row_bytes);
    ln_bulk(mine + k * 2 * row_bytes, x + row * a.ldx, row_bytes, &full[group][k]);
    ln_bulk(mine + k * 2 * row_bytes + row_bytes, dy + row * a.lddy, row_bytes, &full[group][k]);
  };
  if (t == 0)
    for (int k = 0; k < LN_RING - 1; ++k)
      if (first + k * stride < a.n) fill(first + k * stride, k);
  F2 dw[E / 2], db[E / 2];
#pragma unroll
  for (int e = 0; e < E / 2; ++e) dw[e] = db[e] = f2(0.f);
  const float inv_d = 1.f / (float)a.d;
  int turn = 0, k = 0;
  uint32_t phase = 0;
  float next_mu = first < a.n ? a.mean[first] : 0.f, next_rs = first < a.n ? a.rstd[first] : 0.f;
  for (long long row = first; row < a.n; row += stride, turn ^= 1) {
    const float mu = next_mu, rs = next_rs;
    if (row + stride < a.n) {
      next_mu = a.mean[row + stride];
      next_rs = a.rstd[row + stride];
    }
    if (GIVE_UP || !__all_sync(0xffffffffu, mbar_wait(&full[group][k], phase))) {
      ln_bwd_late({full[group], k, LN_RING, LN_RING - 1, phase, row, stride, a.n}, turn, red[group][0], reinterpret_cast<T*>(a.dx), a.d,
                  group, t, threads);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) dw[e] = db[e] = f2(LN_NAN);
      break;
    }
    const uint4 *xs = reinterpret_cast<const uint4*>(mine + k * 2 * row_bytes), *gs = xs + vectors;
    const F2 rs2 = f2(rs), off = f2(-mu);
    F2 s0 = f2(0.f), s1 = f2(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int v = j * threads + t;
      if (v < vectors) {
        Vec<T, V> px, pg;
        px.load(reinterpret_cast<const T*>(xs + v));
        pg.load(reinterpret_cast<const T*>(gs + v));
        F2 w[V / 2];
        ln_get2<V>(w_s, vectors, v, w);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const F2 z = (pair_of(px, i) + off) * rs2, g = pair_of(pg, i), gw = g * w[i];
          dw[j * V / 2 + i] = f2_fma(g, z, dw[j * V / 2 + i]);
          db[j * V / 2 + i] = db[j * V / 2 + i] + g;
          s0 = s0 + gw;
          s1 = f2_fma(gw, z, s1);
        }
      }
    }
    float s[2] = {f2_sum(s0), f2_sum(s1)};
    ln_group_sum<2>(s, red[group][turn], group, t, threads);
    if (threads == 32) __syncwarp();
    if (t == 0 && row + (LN_RING - 1) * stride < a.n) fill(row + (LN_RING - 1) * stride, (k + LN_RING - 1) % LN_RING);
    if (a.dx != nullptr) {
      const F2 mg = f2(-s[0] * inv_d), mgz = f2(-s[1] * inv_d * rs);      // of x - mu
      T* dx = reinterpret_cast<T*>(a.dx) + row * a.d;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int v = j * threads + t;
        if (v < vectors) {
          Vec<T, V> px, pg;
          px.load(reinterpret_cast<const T*>(xs + v));
          pg.load(reinterpret_cast<const T*>(gs + v));
          F2 w[V / 2], o[V / 2];
          ln_get2<V>(w_s, vectors, v, w);
#pragma unroll
          for (int i = 0; i < V / 2; ++i) o[i] = f2_fma(pair_of(px, i) + off, mgz, f2_fma(pair_of(pg, i), w[i], mg)) * rs2;
          store_pairs(dx + v * V, o);
        }
      }
    }
    if (++k == LN_RING) { k = 0; phase ^= 1; }
  }
  if (a.partial == nullptr) return;
  float* acc_s = w_s;
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * a.d; c += blockDim.x) acc_s[c] = 0.f;
  for (int q = 0; q < groups; ++q) {
    __syncthreads();
    if (q != group) continue;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int v = j * threads + t;
      if (v < vectors) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const float2 pw = f2_get(dw[j * V / 2 + i]), pb = f2_get(db[j * V / 2 + i]);
          acc_s[v * V + 2 * i] += pw.x;
          acc_s[v * V + 2 * i + 1] += pw.y;
          acc_s[a.d + v * V + 2 * i] += pb.x;
          acc_s[a.d + v * V + 2 * i + 1] += pb.y;
        }
      }
    }
  }
  __syncthreads();
  float* out = a.partial + (long long)blockIdx.x * 2 * a.d;
  for (int c = threadIdx.x; c < 2 * a.d; c += blockDim.x) out[c] = acc_s[c];
}

template <typename T, int V, int E>
__global__ void __launch_bounds__(1024, 1) ln_bwd_kernel(LnArgs a, int threads, int groups) {
  extern __shared__ float acc_s[];      // [2][D] of the block's groups, added one group after the other
  __shared__ float red[32][2][64];
  const int group = threadIdx.x / threads, t = threadIdx.x % threads;
  pdl_wait();
  pdl_trigger();
  float w[E], dw[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = ln_col<V>(t, threads, e);
    w[e] = c < a.d ? ln_param(a.w, a.w_dt, c, 1.f) : 1.f;
    dw[e] = db[e] = 0.f;
  }
  const float inv_d = 1.f / (float)a.d;
  int turn = 0;
  for (long long row = (long long)blockIdx.x * groups + group; row < a.n; row += (long long)gridDim.x * groups, turn ^= 1) {
    float z[E], g[E];
    ln_load<T, V, E>(reinterpret_cast<const T*>(a.x) + row * a.ldx, a.d, t, threads, z);
    ln_load<T, V, E>(reinterpret_cast<const T*>(a.dy) + row * a.lddy, a.d, t, threads, g);
    const float mu = a.mean[row], rs = a.rstd[row];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      z[e] = (z[e] - mu) * rs;          // columns past D: dy is zero there
      dw[e] = fmaf(g[e], ln_col<V>(t, threads, e) < a.d ? z[e] : 0.f, dw[e]);
      db[e] += g[e];
      g[e] *= w[e];
      s[0] += g[e];
      if (ln_col<V>(t, threads, e) < a.d) s[1] = fmaf(g[e], z[e], s[1]);
    }
    if (a.dx == nullptr) continue;
    ln_group_sum<2>(s, red[group][turn], group, t, threads);
    const float mg = s[0] * inv_d, mgz = s[1] * inv_d;
    T* dx = reinterpret_cast<T*>(a.dx) + row * a.d;
#pragma unroll
    for (int j = 0; j < E / V; ++j) {
      const int c = (j * threads + t) * V;
      if (c >= a.d) continue;
      Vec<T, V> v;
#pragma unroll
      for (int k = 0; k < V; ++k) v.e[k] = from_f<T>(rs * (g[j * V + k] - mg - z[j * V + k] * mgz));
      v.store(dx + c);
    }
  }
  if (a.partial == nullptr) return;
  for (int q = 0; q < groups; ++q) {
    __syncthreads();
    if (q != group) continue;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = ln_col<V>(t, threads, e);
      if (c < a.d) {
        acc_s[c] = (q > 0 ? acc_s[c] : 0.f) + dw[e];
        acc_s[a.d + c] = (q > 0 ? acc_s[a.d + c] : 0.f) + db[e];
      }
    }
  }
  __syncthreads();
  float* out = a.partial + (long long)blockIdx.x * 2 * a.d;
  for (int c = threadIdx.x; c < 2 * a.d; c += blockDim.x) out[c] = acc_s[c];
}

// dw | db: column sums of the partial rows: 32 slices of rows per column (one warp each, all loads under way at once), then the
// slices by a fixed tree
__global__ void __launch_bounds__(1024) ln_reduce_kernel(const float* partial, int blocks, int d, void* dw, void* db, int w_dt) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + lane;
  pdl_wait();
  pdl_trigger();
  float v = 0.f;
  if (c < 2LL * d) {
    const int per = (blocks + 31) / 32, end = min(blocks, (slice + 1) * per);
#pragma unroll 8
    for (int r = slice * per; r < end; ++r) v += partial[(long long)r * 2 * d + c];
  }
  s[slice][lane] = v;
  __syncthreads();
  // warp w sums column w over the slices
  const long long mine = (long long)blockIdx.x * 32 + slice;
  v = ln_warp_sum(s[lane][slice]);
  if (lane != 0 || mine >= 2LL * d) return;
  if (mine < d) {
    if (dw != nullptr) store_any(dw, w_dt, mine, v);
  } else if (db != nullptr) {
    store_any(db, w_dt, mine - d, v);
  }
}

// ---- rows above LN_MAX_ROW elements: one block per row, the row is read again for each pass (it stays in L2) -------
template <typename T>
__global__ void __launch_bounds__(1024) ln_fwd_long_kernel(LnArgs a) {
  __shared__ float red[2][32];
  pdl_wait();
  pdl_trigger();
  const int t = threadIdx.x, nt = blockDim.x;
  for (long long row = blockIdx.x; row < a.n; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
    T* y = reinterpret_cast<T*>(a.y) + row * a.d;
    float s[1] = {0.f};
    for (int c = t; c < a.d; c += nt) s[0] += to_f(x[c]);
    ln_group_sum<1>(s, red[0], 0, t, nt);
    const float mu = s[0] / (float)a.d;
    s[0] = 0.f;
    for (int c = t; c < a.d; c += nt) {
      const float v = to_f(x[c]) - mu;
      s[0] = fmaf(v, v, s[0]);
    }
    ln_group_sum<1>(s, red[1], 0, t, nt);
    const float rs = 1.f / sqrtf(s[0] / (float)a.d + a.eps);
    for (int c = t; c < a.d; c += nt) {
      const float w = a.w != nullptr ? load_any(a.w, a.w_dt, c) : 1.f, b = a.b != nullptr ? load_any(a.b, a.w_dt, c) : 0.f;
      y[c] = from_f<T>(fmaf((to_f(x[c]) - mu) * rs, w, b));
    }
    if (t == 0 && a.mean != nullptr) {
      a.mean[row] = mu;
      a.rstd[row] = rs;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) ln_bwd_long_kernel(LnArgs a) {
  __shared__ float red[2][64];
  pdl_wait();
  pdl_trigger();
  const int t = threadIdx.x, nt = blockDim.x;
  int turn = 0;
  for (long long row = blockIdx.x; row < a.n; row += gridDim.x, turn ^= 1) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = reinterpret_cast<const T*>(a.dy) + row * a.lddy;
    T* dx = reinterpret_cast<T*>(a.dx) + row * a.d;
    const float mu = a.mean[row], rs = a.rstd[row];
    float s[2] = {0.f, 0.f};
    for (int c = t; c < a.d; c += nt) {
      const float g = to_f(dy[c]) * (a.w != nullptr ? load_any(a.w, a.w_dt, c) : 1.f);
      s[0] += g;
      s[1] = fmaf(g, (to_f(x[c]) - mu) * rs, s[1]);
    }
    ln_group_sum<2>(s, red[turn], 0, t, nt);
    const float mg = s[0] / (float)a.d, mgz = s[1] / (float)a.d;
    for (int c = t; c < a.d; c += nt) {
      const float g = to_f(dy[c]) * (a.w != nullptr ? load_any(a.w, a.w_dt, c) : 1.f);
      dx[c] = from_f<T>(rs * (g - mg - (to_f(x[c]) - mu) * rs * mgz));
    }
  }
}

// partial row blockIdx.y: the sums of dy z and dy over the rows blockIdx.y, + gridDim.y, ... of one column per thread
template <typename T>
__global__ void __launch_bounds__(256) ln_wgrad_long_kernel(LnArgs a) {
  pdl_wait();
  pdl_trigger();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.d) return;
  float dw = 0.f, db = 0.f;
  for (long long row = blockIdx.y; row < a.n; row += gridDim.y) {
    const float g = to_f(reinterpret_cast<const T*>(a.dy)[row * a.lddy + c]);
    dw = fmaf(g, (to_f(reinterpret_cast<const T*>(a.x)[row * a.ldx + c]) - a.mean[row]) * a.rstd[row], dw);
    db += g;
  }
  float* out = a.partial + (long long)blockIdx.y * 2 * a.d;
  out[c] = dw;
  out[a.d + c] = db;
}

// ---------------------------------- host side ----------------------------------------------
static std::atomic<int> ln_give_up{0};
// 1: in the launches that follow every row group takes its first wait for one that ran out (for tests of what happens then); returns the state before
extern "C" int layer_norm_give_up(int on) { return ln_give_up.exchange(on); }

// elements per access: as many as the common alignment of all row starts allows
static int ln_vec(const LnArgs& a, int dt, bool bwd) {
  const int es = dt_bytes(dt);
  const uintptr_t bits = bwd ? (uintptr_t)a.x | (uintptr_t)a.dy | (uintptr_t)a.dx | (uintptr_t)(a.ldx * es) |
                                   (uintptr_t)(a.lddy * es) | (uintptr_t)((long long)a.d * es)
                             : (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)(a.ldx * es) | (uintptr_t)((long long)a.d * es);
  if (bits % 16 == 0) return 16 / es;
  return bits % (2 * es) == 0 ? 2 : 1;
}
static int ln_threads(int d, int e) { return ((d + e - 1) / e + 31) / 32 * 32; }

// blocks of the backward kernel = partial rows; one block per SM (its 1024 threads fill the register file)
extern "C" long long layer_norm_partial_floats(int d) { return (long long)sm_count() * 2 * d; }

template <typename T, int V, int NV>
static int ln_launch_fwd(const LnArgs& a, cudaStream_t st) {
  const int threads = 32 * ((a.d + 32 * V * NV - 1) / (32 * V * NV));
  int groups = 256 / threads;
  if (threads > 256) return -1;
  const long long per_sm = (a.n + sm_count() - 1) / sm_count();
  if (groups > per_sm) groups = (int)per_sm;
  long long blocks = (a.n + groups - 1) / groups;
  // as many blocks as the registers of NV vectors leave room for, about
  const long long most = (long long)sm_count() * (NV >= 16 ? 2 : 4) * (256 / (threads * groups));
  if (blocks > most) blocks = most;
  const int smem = 2 * (a.d + V - 1) / V * V * (int)sizeof(float) + 16;
  void (*kernel)(LnArgs, int, int) = ln_fwd_kernel<T, V, NV>;
  if (smem > 40 * 1024) {      // set for every launch: the attribute belongs to the current device
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
  }
  return (int)launch_k(kernel, dim3((unsigned)blocks), dim3((unsigned)(threads * groups)), (size_t)smem, st, a, threads, groups);
}
template <typename T, int NV>
static int ln_launch_fwd_ring(const LnArgs& a, cudaStream_t st, bool* done) {
  constexpr int V = 16 / sizeof(T);
  const int threads = 32 * ((a.d + 32 * V * NV - 1) / (32 * V * NV)), row_bytes = a.d * (int)sizeof(T);
  if (threads > 768) return 0;
  int groups = 768 / threads;
  if (groups > 15 && threads > 32) groups = 15;
  int depth = (int)((215 * 1024 - 8LL * a.d) / ((long long)groups * row_bytes));
  if (depth > 8) depth = 8;
  if (depth < 2) return 0;
  if ((long long)groups * depth * row_bytes > 96 * 1024 && depth > 3) depth = 3;      // about what covers the latency
  *done = true;
  const int smem = 8 * a.d + groups * depth * row_bytes;
  void (*kernel)(LnArgs, int, int, int) = ln_give_up ? ln_fwd_ring_kernel<T, NV, true> : ln_fwd_ring_kernel<T, NV, false>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return (int)e;
  const long long blocks = (a.n + groups - 1) / groups, most = sm_count();
  return (int)launch_k(kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3((unsigned)(threads * groups)), (size_t)smem, st,
                       a, threads, groups, depth);
}
// The ring: rows of at least 2 KB on 16-byte boundaries, enough of them for sixteen groups on every SM, room for two per group.
template <typename T>
static int ln_fwd_ring(const LnArgs& a, cudaStream_t st, bool* done) {
  *done = false;
  if (a.n < 16LL * sm_count() || a.d * (long long)sizeof(T) < 2048) return 0;
  return ln_launch_fwd_ring<T, 4>(a, st, done);
}

// Vectors per lane: 16 when there are rows for eight warps on every SM (a row per warp needs no block barrier), and where the
// row would not fit otherwise; else 4 or 2, so that more warps share a row's latency.
template <typename T, int V>
static int ln_fwd(const LnArgs& a, cudaStream_t st) {
  if (a.d > 256 * V * 4 || (a.n >= 8LL * sm_count() && a.d > 32 * V * 4)) {
    if constexpr (V < 4) {
      if (a.d > 256 * V * 16) return ln_launch_fwd<T, V, 64 / V>(a, st);      // narrow accesses: up to 64 elements per lane
    }
    return ln_launch_fwd<T, V, 16>(a, st);
  }
  if (a.d > 256 * V * 2) return ln_launch_fwd<T, V, 4>(a, st);
  return ln_launch_fwd<T, V, 2>(a, st);
}

// what a call has done: partial rows (blocks of the backward kernel) and launches
struct LnRun {
  int blocks = 0, launches = 0;
};
template <typename T, int V, int E, bool RING>
static int ln_launch_bwd(const LnArgs& a, LnRun* run, cudaStream_t st) {
  const int threads = ln_threads(a.d, E);
  if (threads > 1024) return -1;
  const long long per_sm = (a.n + sm_count() - 1) / sm_count();
  long long groups = (RING && E == 16 ? LN_T16 : 1024) / threads;
  if (groups > 15 && threads > 32) groups = 15;     // named barriers 1 .. 15
  if (RING && groups > 16) groups = 16;
  if (groups > per_sm) groups = per_sm;
  long long smem = (a.partial != nullptr ? 2 : 0) * a.d * (long long)sizeof(float);
  if (RING) {
    const long long stage = 2LL * a.d * (long long)sizeof(T), fixed = (a.d * 8LL + 15) / 16 * 16;
    while (groups > 1 && fixed + groups * LN_RING * stage > 200 * 1024) --groups;
    smem = fixed + groups * LN_RING * stage;
    if (smem > 200 * 1024) return -1;
  }
  long long nb = (a.n + groups - 1) / groups;
  if (nb > sm_count()) nb = sm_count();
  run->blocks = (int)nb;
  void (*kernel)(LnArgs, int, int) = nullptr;
  if constexpr (RING) kernel = ln_give_up ? ln_bwd_ring_kernel<T, E, true> : ln_bwd_ring_kernel<T, E, false>;
  else kernel = ln_bwd_kernel<T, V, E>;
  if (smem > 16 * 1024) {      // set for every launch: the attribute belongs to the current device
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
  }
  return (int)launch_k(kernel, dim3((unsigned)nb), dim3((unsigned)(threads * groups)), (size_t)smem, st, a, threads, (int)groups);
}

template <typename T>
static int ln_dispatch(const LnArgs& a, int dt, bool bwd, LnRun* run, cudaStream_t st) {
  run->launches = 1;
  if (a.d > LN_MAX_ROW) {
    const long long nb = a.n < 2LL * sm_count() ? a.n : 2LL * sm_count();
    if (!bwd) return (int)launch_k(ln_fwd_long_kernel<T>, dim3((unsigned)nb), dim3(1024), 0, st, a);
    if (a.dx != nullptr) {
      int rc = (int)launch_k(ln_bwd_long_kernel<T>, dim3((unsigned)nb), dim3(1024), 0, st, a);
      if (rc) return rc;
    }
    run->launches = (a.dx != nullptr) + (a.partial != nullptr);
    if (a.partial == nullptr) return 0;
    run->blocks = (int)(a.n < 64 ? a.n : 64);
    return (int)launch_k(ln_wgrad_long_kernel<T>, dim3((a.d + 255) / 256, run->blocks), dim3(256), 0, st, a);
  }
  const int v = ln_vec(a, dt, bwd);
  constexpr int W = 16 / sizeof(T);
  if (!bwd) {
    if (v == W) {
      bool done;
      const int rc = ln_fwd_ring<T>(a, st, &done);
      return done || rc ? rc : ln_fwd<T, W>(a, st);
    }
    if (v == 2) return ln_fwd<T, 2>(a, st);
    return ln_fwd<T, 1>(a, st);
  }
  // The ring where its three rows fit, with 8 elements per thread, for 16-bit rows from 1024 on (and for rows above 8192) with
  // 16: half the shuffles per element (16384 x 4096 bf16: 92 against 103 us, 65536 x 1024: 86 against 104).
  if (v == W) {
    if ((long long)a.d * (8 + LN_RING * 2 * (long long)sizeof(T)) <= 200 * 1024 && a.d <= 16 * LN_T16)
      return a.d <= 8192 && (sizeof(T) == 4 || a.d < 1024) ? ln_launch_bwd<T, W, 8, true>(a, run, st)
                                                            : ln_launch_bwd<T, W, 16, true>(a, run, st);
    return a.d <= 8192 ? ln_launch_bwd<T, W, 8, false>(a, run, st) : ln_launch_bwd<T, W, 16, false>(a, run, st);
  }
  if (v == 2) return a.d <= 8192 ? ln_launch_bwd<T, 2, 8, false>(a, run, st) : ln_launch_bwd<T, 2, 16, false>(a, run, st);
  return a.d <= 8192 ? ln_launch_bwd<T, 1, 8, false>(a, run, st) : ln_launch_bwd<T, 1, 16, false>(a, run, st);
}

static int ln_run(const LnArgs& a, int dt, bool bwd, LnRun* run, cudaStream_t st) {
  if (a.n <= 0 || a.d <= 0 || (a.ldx < a.d && a.n > 1 && a.ldx != 0) || a.w_dt < 0 || a.w_dt > 2) return -1;
  if (dt == DT_F32) return ln_dispatch<float>(a, dt, bwd, run, st);
  if (dt == DT_BF16) return ln_dispatch<__nv_bfloat16>(a, dt, bwd, run, st);
  if (dt == DT_F16) return ln_dispatch<__half>(a, dt, bwd, run, st);
  return -1;
}

extern "C" int layer_norm_forward(LnForwardCall* c) {
  LnArgs a = {};
  a.x = c->x; a.w = c->w; a.b = c->b; a.y = c->y; a.n = c->n; a.ldx = c->ldx; a.d = (int)c->d; a.eps = (float)c->eps;
  a.w_dt = (int)c->w_dt;
  a.mean = c->stats;
  a.rstd = c->stats != nullptr ? c->stats + c->n : nullptr;
  LnRun run;
  const int rc = ln_run(a, (int)c->dt, false, &run, (cudaStream_t)c->stream);
  c->launches = run.launches;
  return rc;
}

extern "C" int layer_norm_backward(LnBackwardCall* c) {
  if ((c->dw != nullptr || c->db != nullptr) != (c->partial != nullptr)) return -1;
  LnArgs a = {};
  a.x = c->x; a.dy = c->dy; a.lddy = c->lddy; a.w = c->w; a.mean = c->stats; a.rstd = c->stats + c->n;
  a.dx = c->dx; a.partial = c->partial; a.n = c->n; a.ldx = c->ldx; a.d = (int)c->d; a.w_dt = (int)c->w_dt;
  LnRun run;
  const int rc = ln_run(a, (int)c->dt, true, &run, (cudaStream_t)c->stream);
  c->launches = run.launches + (c->partial != nullptr);
  if (rc || c->partial == nullptr) return rc;
  // a programmatic dependent of the kernel before (1120 x 650 fp32, the whole training pass: 16.4 -> 15.7 us)
  return (int)launch_k_if(pdl_in_call() || pdl_enabled(), ln_reduce_kernel, dim3((unsigned)((2LL * a.d + 31) / 32)), dim3(1024), 0, (cudaStream_t)c->stream,
                       (const float*)c->partial, run.blocks, a.d, c->dw, c->db, a.w_dt);
}

// 0, or 1 after a bounded wait of a kernel on the current device ran out since the last call (synchronises)
extern "C" int layer_norm_last_error() {
  int v = -1;
  if (cudaMemcpyFromSymbol(&v, g_ln_error, sizeof(int)) != cudaSuccess) return -1;
  const int none = 0;
  if (v != 0) cudaMemcpyToSymbol(g_ln_error, &none, sizeof(int));
  return v;
}
