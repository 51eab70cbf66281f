// Layer normalisation over the last dimension (width D) of an [N, D] matrix, forward and backward.
//
//   mu = mean(x), var = mean((x - mu)^2), rs = 1 / sqrt(var + eps), z = (x - mu) rs, y = z w + b
//   g = dy w;  dx = rs (g - mean(g) - z mean(g z));  dw = sum over rows of dy z;  db = sum over rows of dy
//
// Both directions are one pass over memory: a row is read once, held in registers (the variance is taken about the
// mean, not from a sum of squares) and written once.  A row belongs to a group of T = 32 .. 1024 threads with E = 8
// consecutive-vector elements each (16 for rows above 8192); a block holds several groups and walks over the rows, so
// that weight and bias are fetched once per block.  All statistics and sums are fp32.
//
// The backward kernel keeps the running sums of dw and db of its columns in registers over all rows of its block,
// adds the block's groups in shared memory and writes one partial row per block; a second kernel adds the partial
// rows in block order.  No atomics: the same inputs give the same bits.
//
// Rows that do not start on 16-byte (8- / 4-byte) boundaries take narrower accesses (V elements at a time); rows
// too long for registers (above 16384 elements) take the *_long kernels, which read the row again from L2.
#include "launch.cuh"
#include "vec.cuh"

#define LN_MAX_ROW 16384

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

template <typename T, int V, int E>
__global__ void __launch_bounds__(1024) ln_fwd_kernel(LnArgs a, int threads, int groups) {
  __shared__ float red[32][2][32];   // [group][buffer][warp]
  const int group = threadIdx.x / threads, t = threadIdx.x % threads;
  pdl_wait();
  pdl_trigger();
  float w[E], b[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = ln_col<V>(t, threads, e);
    w[e] = c < a.d && a.w != nullptr ? load_any(a.w, a.w_dt, c) : 1.f;
    b[e] = c < a.d && a.b != nullptr ? load_any(a.b, a.w_dt, c) : 0.f;
  }
  const float inv_d = 1.f / (float)a.d;
  for (long long row = (long long)blockIdx.x * groups + group; row < a.n; row += (long long)gridDim.x * groups) {
    float x[E];
    ln_load<T, V, E>(reinterpret_cast<const T*>(a.x) + row * a.ldx, a.d, t, threads, x);
    float s[1] = {0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) s[0] += x[e];
    ln_group_sum<1>(s, red[group][0], group, t, threads);
    const float mu = s[0] * inv_d;
    s[0] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x[e] -= mu;
      if (ln_col<V>(t, threads, e) < a.d) s[0] = fmaf(x[e], x[e], s[0]);
    }
    ln_group_sum<1>(s, red[group][1], group, t, threads);
    const float rs = 1.f / sqrtf(fmaf(s[0], inv_d, a.eps));
    T* y = reinterpret_cast<T*>(a.y) + row * a.d;
#pragma unroll
    for (int j = 0; j < E / V; ++j) {
      const int c = (j * threads + t) * V;
      if (c >= a.d) continue;
      Vec<T, V> v;
#pragma unroll
      for (int k = 0; k < V; ++k) v.e[k] = from_f<T>(fmaf(x[j * V + k] * rs, w[j * V + k], b[j * V + k]));
      v.store(y + c);
    }
    if (t == 0 && a.mean != nullptr) {
      a.mean[row] = mu;
      a.rstd[row] = rs;
    }
  }
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
    w[e] = c < a.d && a.w != nullptr ? load_any(a.w, a.w_dt, c) : 1.f;
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

// dw | db: column sums of the partial rows in block order; eight slices of rows per column, then the slices in order
__global__ void __launch_bounds__(256) ln_reduce_kernel(const float* partial, int blocks, int d, void* dw, void* db, int w_dt) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + lane;
  pdl_wait();
  pdl_trigger();
  float v = 0.f;
  if (c < 2 * d) {
    const int per = (blocks + 7) / 8, end = min(blocks, (slice + 1) * per);
    for (int r = slice * per; r < end; ++r) v += partial[(long long)r * 2 * d + c];
  }
  s[slice][lane] = v;
  __syncthreads();
  if (slice != 0 || c >= 2 * d) return;
  v = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) v += s[k][lane];
  if (c < d) {
    if (dw != nullptr) store_any(dw, w_dt, c, v);
  } else if (db != nullptr) {
    store_any(db, w_dt, c - d, v);
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

template <typename T, int V, int E>
static int ln_launch(const LnArgs& a, bool bwd, int* blocks, cudaStream_t st) {
  const int threads = ln_threads(a.d, E);
  const long long per_sm = (a.n + sm_count() - 1) / sm_count();
  if (!bwd) {
    // groups per block: about 256 threads, fewer when there are too few rows to give every SM a block
    long long groups = threads >= 256 ? 1 : 256 / threads;
    if (groups > per_sm) groups = per_sm;
    long long blocks_f = (a.n + groups - 1) / groups;
    const long long most = (long long)sm_count() * (2048 / (threads * groups < 32 ? 32 : threads * groups));
    if (blocks_f > most) blocks_f = most;
    return (int)launch_k(ln_fwd_kernel<T, V, E>, dim3((unsigned)blocks_f), dim3((unsigned)(threads * groups)), 0, st, a,
                         threads, (int)groups);
  }
  long long groups = 1024 / threads;
  if (groups > 15 && threads > 32) groups = 15;     // named barriers 1 .. 15
  if (groups > per_sm) groups = per_sm;
  long long nb = (a.n + groups - 1) / groups;
  if (nb > sm_count()) nb = sm_count();
  *blocks = (int)nb;
  const int smem = a.partial != nullptr ? 2 * a.d * (int)sizeof(float) : 0;
  if (smem > 32 * 1024) {
    // set for every launch: the attribute belongs to the current device
    cudaError_t e = cudaFuncSetAttribute(ln_bwd_kernel<T, V, E>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
  }
  return (int)launch_k(ln_bwd_kernel<T, V, E>, dim3((unsigned)nb), dim3((unsigned)(threads * groups)), (size_t)smem, st,
                       a, threads, (int)groups);
}

template <typename T>
static int ln_dispatch(const LnArgs& a, int dt, bool bwd, int* blocks, cudaStream_t st) {
  if (a.d > LN_MAX_ROW) {
    const long long nb = a.n < 2LL * sm_count() ? a.n : 2LL * sm_count();
    if (!bwd) return (int)launch_k(ln_fwd_long_kernel<T>, dim3((unsigned)nb), dim3(1024), 0, st, a);
    if (a.dx != nullptr) {
      int rc = (int)launch_k(ln_bwd_long_kernel<T>, dim3((unsigned)nb), dim3(1024), 0, st, a);
      if (rc) return rc;
    }
    *blocks = 0;
    if (a.partial == nullptr) return 0;
    *blocks = (int)(a.n < 64 ? a.n : 64);
    return (int)launch_k(ln_wgrad_long_kernel<T>, dim3((a.d + 255) / 256, *blocks), dim3(256), 0, st, a);
  }
  const int v = ln_vec(a, dt, bwd);
  constexpr int W = 16 / sizeof(T);
  if (a.d <= 8192) {
    if (v == W) return ln_launch<T, W, 8>(a, bwd, blocks, st);
    if (v == 2) return ln_launch<T, 2, 8>(a, bwd, blocks, st);
    return ln_launch<T, 1, 8>(a, bwd, blocks, st);
  }
  if (v == W) return ln_launch<T, W, 16>(a, bwd, blocks, st);
  if (v == 2) return ln_launch<T, 2, 16>(a, bwd, blocks, st);
  return ln_launch<T, 1, 16>(a, bwd, blocks, st);
}

static int ln_run(const LnArgs& a, int dt, bool bwd, int* blocks, cudaStream_t st) {
  if (a.n <= 0 || a.d <= 0 || (a.ldx < a.d && a.n > 1 && a.ldx != 0) || a.w_dt < 0 || a.w_dt > 2) return -1;
  if (dt == DT_F32) return ln_dispatch<float>(a, dt, bwd, blocks, st);
  if (dt == DT_BF16) return ln_dispatch<__nv_bfloat16>(a, dt, bwd, blocks, st);
  if (dt == DT_F16) return ln_dispatch<__half>(a, dt, bwd, blocks, st);
  return -1;
}

// y = layer_norm(x) w + b; mean / rstd may be null (evaluation)
extern "C" int layer_norm_forward(const void* x, long long ldx, const void* w, const void* b, void* y, float* mean,
                                  float* rstd, long long n, int d, float eps, int dt, int w_dt, cudaStream_t st) {
  LnArgs a = {};
  a.x = x; a.w = w; a.b = b; a.y = y; a.mean = mean; a.rstd = rstd; a.n = n; a.ldx = ldx; a.d = d; a.eps = eps; a.w_dt = w_dt;
  int blocks = 0;
  return ln_run(a, dt, false, &blocks, st);
}

// dx (may be null) and dw, db (may be null; partial: layer_norm_partial_floats(d) floats of scratch, or null without both)
extern "C" int layer_norm_backward(const void* x, long long ldx, const void* dy, long long lddy, const void* w,
                                   const float* mean, const float* rstd, void* dx, void* dw, void* db, float* partial,
                                   long long n, int d, int dt, int w_dt, cudaStream_t st) {
  if ((dw != nullptr || db != nullptr) != (partial != nullptr)) return -1;
  LnArgs a = {};
  a.x = x; a.dy = dy; a.lddy = lddy; a.w = w; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.dx = dx; a.partial = partial; a.n = n; a.ldx = ldx; a.d = d; a.w_dt = w_dt;
  int blocks = 0;
  int rc = ln_run(a, dt, true, &blocks, st);
  if (rc || partial == nullptr) return rc;
  return (int)launch_k(ln_reduce_kernel, dim3((unsigned)((2LL * d + 31) / 32)), dim3(256), 0, st, (const float*)partial,
                       blocks, d, dw, db, w_dt);
}
