// Gated feed-forward block for few tokens (evaluation): one pass over the weights, no tensor core.
//
//   h[m, f] = act(x[m] . W_in[f]) (x[m] . W_in[F + f])          y[m, n] = h[m] . W_out[n]
//
// Bound by reading the weights once.  The columns of the result are dealt out evenly over the blocks; a warp takes four weight
// rows at a time (two gate rows and their up rows, or four rows of W_out) and a slice of k, 16 bytes per lane, row and step,
// and multiplies them with all tokens, whose values come from L1 once per four rows.  fp32 multiply-adds and sums, h in fp32.
// The lanes' sums of 32 values are brought together in 31 shuffles (each step halves the number of values a lane holds);
// the warps of a k split meet in shared memory.  Fixed order: the same inputs give the same bits.
//
// Tokens: up to 4 for 16-bit weights, up to 8 for fp32.  Above, the multiply-adds (tokens per weight) take longer than the weights'
// way from memory: 16-bit operands then go to the tensor core (2048 x 8192 bf16, this form against the tensor-core form: 1 token
// 23 / 36 us, 4 tokens 33 / 37, 8 tokens 60 / 35); fp32, whose tensor-core form has to split the weights first, takes tiles of 32
// tokens x 32 weight rows on the fp32 units up to 32 tokens (ffn_tile_kernel; 2048 x 8192: 16 tokens 123 / 165 us, 32 tokens
// 125 / 165, 48 tokens 232 / 166).
#include "ffn.cuh"
#include "launch.cuh"

#define FEW_THREADS 256
#define FEW_WARPS 8
#define FEW_ROWS 4          // weight rows of a warp

struct FewArgs {
  const void* w;
  const void* x;
  void* out;
  long long ldw, up, ldx, ldo;     // up: elements from a gate row to its up row
  int m, n, k, act, k_split;       // k_split: warps that share a row (power of two)
};

template <typename T, int V>
__device__ __forceinline__ void few_load(const T* p, float* f) {
  if (sizeof(T) * V == 32) {       // eight floats: two accesses
    Vec<T, 16 / sizeof(T)> a, b;
    a.load(p);
    b.load(p + 16 / sizeof(T));
#pragma unroll
    for (int e = 0; e < 16 / (int)sizeof(T); ++e) {
      f[e] = to_f(a.e[e]);
      f[e + 16 / sizeof(T)] = to_f(b.e[e]);
    }
  } else {
    Vec<T, (sizeof(T) * V > 16 ? 16 / sizeof(T) : V)> a;
    a.load(p);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = to_f(a.e[e]);
  }
}

// lane l ends with the sum over all lanes of value l (N = 32), or of value l / (32 / N)
template <int N>
__device__ __forceinline__ float few_reduce(float* v, int lane) {
  int n = N;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (n > 1) {
      n >>= 1;
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        if (i < n) {
          const float give = (lane & o) ? v[i] : v[i + n], keep = (lane & o) ? v[i + n] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
  return v[0];
}

// TW weights, TX the other factor, TO results; MT tokens (a.m <= MT), V elements per access
template <typename TW, typename TX, typename TO, int MT, int V, bool GATE>
__global__ void __launch_bounds__(FEW_THREADS) ffn_few_kernel(FewArgs a) {
  constexpr int RG = GATE ? FEW_ROWS / 2 : FEW_ROWS;     // result columns of a warp
  constexpr int NV = FEW_ROWS * MT;
  __shared__ float sums[2][FEW_WARPS][NV];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ks = warp & (a.k_split - 1), group = warp / a.k_split, groups = FEW_WARPS / a.k_split;
  const int all = (a.n + RG - 1) / RG;       // groups of result columns, dealt out to the blocks
  const int c0 = (int)((long long)all * blockIdx.x / gridDim.x) * RG;
  const int c1 = min(a.n, (int)((long long)all * (blockIdx.x + 1) / gridDim.x) * RG);
  const int steps = (a.k + 32 * V - 1) / (32 * V);
  const int s0 = (int)((long long)steps * ks / a.k_split), s1 = (int)((long long)steps * (ks + 1) / a.k_split);
  const TW* w = reinterpret_cast<const TW*>(a.w);
  const TX* x = reinterpret_cast<const TX*>(a.x);
  int turn = 0;
  for (int base = c0; base < c1; base += RG * groups, turn ^= 1) {
    const int col = base + group * RG;
    if (col < c1) {
      const TW* row[FEW_ROWS];
#pragma unroll
      for (int j = 0; j < FEW_ROWS; ++j) {
        const int c = min(col + (GATE ? j % RG : j), c1 - 1);        // past the block's columns: the last one again, not stored
        row[j] = w + (long long)c * a.ldw + (GATE && j >= RG ? a.up : 0);
      }
      float acc[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) acc[i] = 0.f;
      const auto step = [&](int k) {
        float wv[FEW_ROWS][V];
#pragma unroll
        for (int j = 0; j < FEW_ROWS; ++j) few_load<TW, V>(row[j] + k, wv[j]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          float xv[V];
          few_load<TX, V>(x + (long long)min(m, a.m - 1) * a.ldx + k, xv);
#pragma unroll
          for (int j = 0; j < FEW_ROWS; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) acc[j * MT + m] = fmaf(wv[j][e], xv[e], acc[j * MT + m]);
        }
      };
      // whole steps have no condition, so that the loads of several are under way at once
      const int whole = min(s1, a.k / (32 * V));
#pragma unroll (MT <= 4 ? 4 : 2)
      for (int s = s0; s < whole; ++s) step((s * 32 + lane) * V);
      if (whole < s1 && (whole * 32 + lane) * V < a.k) step((whole * 32 + lane) * V);
      constexpr int N = NV < 32 ? NV : 32;
#pragma unroll
      for (int q = 0; q < NV; q += N) {
        const float v = few_reduce<N>(acc + q, lane);
        if (lane % (32 / N) == 0) sums[turn][warp][q + lane / (32 / N)] = v;
      }
    }
    __syncthreads();
    if (ks == 0 && col < c1) {
#pragma unroll
      for (int t = lane; t < RG * MT; t += 32) {
        const int j = t / MT, m = t % MT;
        if (col + j < c1 && m < a.m) {
          float v = 0.f, u = 0.f;
          for (int q = 0; q < a.k_split; ++q) {
            v += sums[turn][warp + q][j * MT + m];
            if (GATE) u += sums[turn][warp + q][(RG + j) * MT + m];
          }
          if (GATE) {
            constexpr bool FAST = sizeof(TW) == 2;
            float slope, h;
            if (a.act == ACT_SILU) h = ff_act<ACT_SILU, false, FAST>(v, slope);
            else if (a.act == ACT_GELU) h = ff_act<ACT_GELU, false, FAST>(v, slope);
            else if (a.act == ACT_RELU) h = ff_act<ACT_RELU, false, FAST>(v, slope);
            else h = ff_act<ACT_SIGMOID, false, FAST>(v, slope);
            v = h * u;
          }
          reinterpret_cast<TO*>(a.out)[(long long)m * a.ldo + col + j] = from_f<TO>(v);
        }
      }
    }
  }
}

// Blocks: as many as fit on an SM by their registers (four, two), fewer for few columns.  Warps per row (k_split): the
// cheapest by  rounds of a block x (steps x cycles of a step + cycles of bringing the sums together), with two to eight warps
// on a scheduler.
template <typename TW, typename TX, typename TO, int MT, int V, bool GATE>
static int few_launch(FewArgs& a, cudaStream_t st) {
  constexpr int RG = GATE ? FEW_ROWS / 2 : FEW_ROWS;
  const int most = sm_count() * (MT >= 8 ? 2 : 4), cols = (a.n + RG - 1) / RG;
  const int grid = cols < most ? cols : most;
  const int groups = (cols + grid - 1) / grid, steps = (a.k + 32 * V - 1) / (32 * V);
  const int step = 8 * MT * V > 100 ? 8 * MT * V : 100, join = 100 + 24 * MT;
  long long best = 1LL << 62;
  for (int q = 1; q <= FEW_WARPS && q <= steps; q *= 2) {
    const int wr = FEW_WARPS / q;
    const long long cost = (long long)((groups + wr - 1) / wr) * ((long long)((steps + q - 1) / q) * step + join);
    if (cost < best) { best = cost; a.k_split = q; }
  }
  return (int)launch_k(ffn_few_kernel<TW, TX, TO, MT, V, GATE>, dim3(grid), dim3(FEW_THREADS), 0, st, a);
}
template <typename TW, typename TX, typename TO, int V, bool GATE>
static int few_tokens(FewArgs& a, cudaStream_t st) {
  if (a.m <= 1) return few_launch<TW, TX, TO, 1, V, GATE>(a, st);
  if (a.m <= 2) return few_launch<TW, TX, TO, 2, V, GATE>(a, st);
  if (a.m <= 4) return few_launch<TW, TX, TO, 4, V, GATE>(a, st);
  if constexpr (sizeof(TW) == 4) {
    if (a.m <= 8) return few_launch<TW, TX, TO, 8, V, GATE>(a, st);
  }
  return -1;
}
// V: the widest access that all rows of both factors and k allow
template <typename T, typename TX, typename TO, bool GATE>
static int few_width(FewArgs& a, cudaStream_t st) {
  constexpr int W = 16 / (int)sizeof(T);
  const auto fits = [&](int v) {
    const long long wb = v * (long long)sizeof(T), xb = v * (long long)sizeof(TX) > 16 ? 16 : v * (long long)sizeof(TX);
    return a.k % v == 0 && (uintptr_t)a.w % wb == 0 && a.ldw * (long long)sizeof(T) % wb == 0 &&
           (!GATE || a.up * (long long)sizeof(T) % wb == 0) && (uintptr_t)a.x % xb == 0 && a.ldx * (long long)sizeof(TX) % xb == 0;
  };
  if (fits(W)) return few_tokens<T, TX, TO, W, GATE>(a, st);
  if (fits(2)) return few_tokens<T, TX, TO, 2, GATE>(a, st);
  return few_tokens<T, TX, TO, 1, GATE>(a, st);
}
template <typename T>
static int few_forward(FewArgs& in, FewArgs& out, cudaStream_t st) {
  const int rc = few_width<T, T, float, true>(in, st);
  return rc ? rc : few_width<T, float, T, false>(out, st);
}

// ---- fp32, 9 to 32 tokens ------------------------------------------------------------------------------------------
// A block multiplies 32 tokens with 32 weight rows (gate: 16 gate rows and their up rows).  64 k at a time come into shared
// memory by cp.async (four stages); four groups of 64 threads take 16 k each, a thread 4 tokens x 4 rows (8 loads of 16 bytes
// from shared memory for 64 multiply-adds).  The groups' sums, then those of the blocks of a cluster, which share a long k
// (W_out's products have few rows), are added in a fixed order.
#define FT_K 64
#define FT_LD (FT_K + 4)             // floats per row: eight rows read at once fall into different banks
#define FT_STAGES 4
#define FT_SMEM (FT_STAGES * 2 * 32 * FT_LD * 4)

template <int V>
__device__ __forceinline__ void ft_copy(float* dst, const float* src, bool inside) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst), n = inside ? 4 * V : 0;     // 0: the destination is zeroed
  if (V == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
  else if (V == 2) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
}

template <int V, bool GATE>
__global__ void __launch_bounds__(256) ffn_tile_kernel(FewArgs a) {
  extern __shared__ float4 ft_smem4[];
  float* smem = reinterpret_cast<float*>(ft_smem4);
  pdl_wait();
  pdl_trigger();
  const int t = threadIdx.x, slices = a.k_split;        // blocks of a cluster
  const int slice = (int)(blockIdx.x % slices), c0 = (int)(blockIdx.x / slices) * (GATE ? 16 : 32);
  const int steps = (a.k + FT_K - 1) / FT_K;
  const int s0 = (int)((long long)steps * slice / slices), s1 = (int)((long long)steps * (slice + 1) / slices);
  const float *w = reinterpret_cast<const float*>(a.w), *x = reinterpret_cast<const float*>(a.x);
  // a thread copies V floats at column k0 of every (256 V / 64)-th of the 64 rows (32 of weights, 32 of tokens)
  constexpr int RS = 256 / (FT_K / V), NR = 64 / RS;
  const int k0 = t % (FT_K / V) * V, r0 = t / (FT_K / V);
  const float* src[NR];
  uint32_t rows = 0;               // bit j: row j exists
#pragma unroll
  for (int j = 0; j < NR; ++j) {
    const int r = r0 + RS * j;
    bool inside;
    if (r < 32) {
      const int c = c0 + (GATE ? (r & 15) : r);
      inside = c < a.n;
      src[j] = w + (inside ? (long long)c * a.ldw + (GATE && r >= 16 ? a.up : 0) : 0) + k0;
    } else {
      inside = r - 32 < a.m;
      src[j] = x + (inside ? (long long)(r - 32) * a.ldx : 0) + k0;
    }
    rows |= (uint32_t)inside << j;
  }
  const auto fetch = [&](int s) {
    float* stage = smem + (s - s0) % FT_STAGES * (2 * 32 * FT_LD) + r0 * FT_LD + k0;
    const bool in_k = s * FT_K + k0 < a.k;
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      const bool inside = in_k && (rows >> j & 1u);
      ft_copy<V>(stage + j * RS * FT_LD, inside ? src[j] + s * FT_K : (j * RS + r0 < 32 ? w : x), inside);
    }
  };
#pragma unroll
  for (int s = 0; s < FT_STAGES - 1; ++s) {
    if (s0 + s < s1) fetch(s0 + s);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  const int kg = t >> 6, tg = t & 7, rg = (t >> 3) & 7;
  float acc[4][4] = {};            // [row rg + 8 i][token tg + 8 j]
  for (int s = s0; s < s1; ++s) {
    asm volatile("cp.async.wait_group %0;" ::"n"(FT_STAGES - 2) : "memory");
    __syncthreads();               // the stage is complete, and the one that is fetched next has been read by everyone
    if (s + FT_STAGES - 1 < s1) fetch(s + FT_STAGES - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    const float* sw = smem + (s - s0) % FT_STAGES * (2 * 32 * FT_LD) + kg * 16;
    const float* sx = sw + 32 * FT_LD;
#pragma unroll
    for (int k = 0; k < 16; k += 4) {
      float4 p[4], q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = *reinterpret_cast<const float4*>(sw + (rg + 8 * i) * FT_LD + k);
        q[i] = *reinterpret_cast<const float4*>(sx + (tg + 8 * i) * FT_LD + k);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = fmaf(p[i].x, q[j].x, acc[i][j]);
          acc[i][j] = fmaf(p[i].y, q[j].y, acc[i][j]);
          acc[i][j] = fmaf(p[i].z, q[j].z, acc[i][j]);
          acc[i][j] = fmaf(p[i].w, q[j].w, acc[i][j]);
        }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  // sums [group][row][token], 33 floats per row
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) smem[(kg * 32 + rg + 8 * i) * 33 + tg + 8 * j] = acc[i][j];
  __syncthreads();
  float* total = smem + 4 * 32 * 33;
  for (int i = t; i < 1024; i += 256) {
    const int r = i >> 5, m = i & 31;
    float v = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g) v += smem[(g * 32 + r) * 33 + m];
    total[r * 33 + m] = v;
  }
  if (slices > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else __syncthreads();
  const uint32_t mine = (uint32_t)__cvta_generic_to_shared(total);
  // of a cluster, every block writes its share of the results; consecutive threads take consecutive columns of a token
  constexpr int OUT = GATE ? 512 : 1024, COLS = GATE ? 16 : 32;
  for (int i = slice * 256 + t; i < OUT; i += slices * 256) {
    const int r = i % COLS, m = i / COLS;
    float v = 0.f, u = 0.f;
    for (int q = 0; q < slices; ++q) {
      float p, z = 0.f;
      uint32_t at;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(mine), "r"(q));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(p) : "r"(at + (r * 33 + m) * 4) : "memory");
      if (GATE) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(z) : "r"(at + ((r + 16) * 33 + m) * 4) : "memory");
      v += p;
      u += z;
    }
    if (c0 + r < a.n && m < a.m) {
      if (GATE) {
        float slope, h;
        if (a.act == ACT_SILU) h = ff_act<ACT_SILU, false, false>(v, slope);
        else if (a.act == ACT_GELU) h = ff_act<ACT_GELU, false, false>(v, slope);
        else if (a.act == ACT_RELU) h = ff_act<ACT_RELU, false, false>(v, slope);
        else h = ff_act<ACT_SIGMOID, false, false>(v, slope);
        v = h * u;
      }
      reinterpret_cast<float*>(a.out)[(long long)m * a.ldo + c0 + r] = v;
    }
  }
  // the other blocks have read this one's sums
  if (slices > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int V, bool GATE>
static int ft_launch(FewArgs& a, cudaStream_t st) {
  void (*kernel)(FewArgs) = ffn_tile_kernel<V, GATE>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FT_SMEM);
  if (e != cudaSuccess) return (int)e;
  const int tiles = (a.n + (GATE ? 15 : 31)) / (GATE ? 16 : 32), steps = (a.k + FT_K - 1) / FT_K;
  a.k_split = 1;
  // slices of k: the cheapest by  blocks per SM x (steps + what a block costs besides, about two steps)
  long long best = 1LL << 62;
  for (int q = 1; q <= 8 && q <= steps; q *= 2) {
    const long long cost = (long long)((tiles * (long long)q + sm_count() - 1) / sm_count()) * ((steps + q - 1) / q + 2);
    if (cost < best) { best = cost; a.k_split = q; }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * a.k_split));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = FT_SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (a.k_split > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = a.k_split;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return (int)cudaLaunchKernelEx(&cfg, kernel, a);
}
template <bool GATE>
static int ft_width(FewArgs& a, cudaStream_t st) {
  const auto fits = [&](int v) {
    return a.k % v == 0 && ((uintptr_t)a.w | (uintptr_t)a.x | (uintptr_t)(a.ldw * 4) | (uintptr_t)(a.ldx * 4) | (uintptr_t)(a.up * 4)) % (4 * v) == 0;
  };
  if (fits(4)) return ft_launch<4, GATE>(a, st);
  if (fits(2)) return ft_launch<2, GATE>(a, st);
  return ft_launch<1, GATE>(a, st);
}

int ffn_few_tokens(int dt) { return dt == DT_F32 ? 32 : 4; }

int ffn_few_forward(const void* x, long long ldx, const void* w_in, long long ld_in, const void* w_out, long long ld_out, float* h,
                    void* y, int m, int d, int f, int n, int act, int dt, cudaStream_t st) {
  if (m > ffn_few_tokens(dt)) return -1;
  const long long ldh = (f + 15) / 16 * 16;
  FewArgs in = {w_in, x, h, ld_in, (long long)f * ld_in, ldx, ldh, m, f, d, act, 1};
  FewArgs out = {w_out, h, y, ld_out, 0, ldh, n, m, n, f, act, 1};
  if (dt == DT_F32 && m > 8) {
    const int rc = ft_width<true>(in, st);
    return rc ? rc : ft_width<false>(out, st);
  }
  if (dt == DT_F32) return few_forward<float>(in, out, st);
  if (dt == DT_BF16) return few_forward<__nv_bfloat16>(in, out, st);
  return few_forward<__half>(in, out, st);
}
