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
// Tokens: 16-bit weights up to 8, fp32 up to 32.  Above, the multiply-adds (tokens per weight) take longer than the weights' way
// from memory, and the tensor-core form is faster.
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
#pragma unroll (MT <= 4 ? 4 : (MT <= 8 ? 2 : 1))
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

// Blocks: as many as fit on an SM by their registers (four, two, one), fewer for few columns.  Warps per row (k_split): the
// cheapest by  rounds of a block x (steps x cycles of a step + cycles of bringing the sums together), with two to eight warps
// on a scheduler.
template <typename TW, typename TX, typename TO, int MT, int V, bool GATE>
static int few_launch(FewArgs& a, cudaStream_t st) {
  constexpr int RG = GATE ? FEW_ROWS / 2 : FEW_ROWS;
  const int most = sm_count() * (MT >= 16 ? 1 : (MT >= 8 ? 2 : 4)), cols = (a.n + RG - 1) / RG;
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
  if (a.m <= 4) return few_launch<TW, TX, TO, 4, V, GATE>(a, st);
  if (a.m <= 8) return few_launch<TW, TX, TO, 8, V, GATE>(a, st);
  if constexpr (sizeof(TW) == 4) {
    if (a.m <= 16) return few_launch<TW, TX, TO, 16, V, GATE>(a, st);
    if (a.m <= 32) return few_launch<TW, TX, TO, 32, V, GATE>(a, st);
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

int ffn_few_tokens(int dt) { return dt == DT_F32 ? 32 : 8; }

int ffn_few_forward(const void* x, long long ldx, const void* w_in, long long ld_in, const void* w_out, long long ld_out, float* h,
                    void* y, int m, int d, int f, int n, int act, int dt, cudaStream_t st) {
  if (m > ffn_few_tokens(dt)) return -1;
  const long long ldh = (f + 15) / 16 * 16;
  FewArgs in = {w_in, x, h, ld_in, (long long)f * ld_in, ldx, ldh, m, f, d, act, 1};
  FewArgs out = {w_out, h, y, ld_out, 0, ldh, n, m, n, f, act, 1};
  if (dt == DT_F32) return few_forward<float>(in, out, st);
  if (dt == DT_BF16) return few_forward<__nv_bfloat16>(in, out, st);
  return few_forward<__half>(in, out, st);
}
