// Gated feed-forward block for few tokens (evaluation): one pass over the weights as they lie in memory.
//
//   h[m, f] = act(x[m] . W_in[f]) (x[m] . W_in[F + f])          y[m, n] = h[m] . W_out[n]
//
// Bound by reading the weights once.  Up to 4 tokens (fp32: 8) the columns of the result are dealt out evenly over the blocks; a
// warp takes four weight rows at a time (two gate rows and their up rows, or four rows of W_out) and a slice of k, 16 bytes per
// lane, row and step, and multiplies them with all tokens, whose values come from L1 once per four rows.  fp32 multiply-adds and
// sums, h in fp32.  The lanes' sums of 32 values are brought together in 31 shuffles (each step halves the number of values a lane
// holds); the warps of a k split meet in shared memory.  Fixed order: the same inputs give the same bits.
//
// Above, the multiply-adds (tokens per weight) take longer than the weights' way from memory (2048 x 8192 bf16: 1 token 22 us,
// 4 tokens 33, 8 tokens 60), and the products go to the warps' matrix instruction (ffn_mma_kernel): fp32 up to 32 tokens, which
// saves the tensor-core form's pass that splits the weights (32 tokens, this form / that one: 650 x 2600 26 / 39 us, 2048 x 8192
// 93 / 166; 48 tokens 43 / 39 and 195 / 166); 16 bits up to 16 tokens and 2^25 weights, where that form's setup counts
// (16 tokens: 650 x 2600 14 / 21, 1536 x 6144 25 / 29, 2048 x 8192 39 / 36; 32 tokens: 20 / 21, 32 / 28, 53 / 32).
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

template <bool FAST>
__device__ __forceinline__ float few_act(int act, float z) {
  float slope;
  if (act == ACT_SILU) return ff_act<ACT_SILU, false, FAST>(z, slope);
  if (act == ACT_GELU) return ff_act<ACT_GELU, false, FAST>(z, slope);
  if (act == ACT_RELU) return ff_act<ACT_RELU, false, FAST>(z, slope);
  return ff_act<ACT_SIGMOID, false, FAST>(z, slope);
}

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
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ks = warp & (a.k_split - 1), group = warp / a.k_split, groups = FEW_WARPS / a.k_split;
  const int all = (a.n + RG - 1) / RG;       // groups of result columns, dealt out to the blocks
  const int c0 = (int)((long long)all * blockIdx.x / gridDim.x) * RG;
  const int c1 = min(a.n, (int)((long long)all * (blockIdx.x + 1) / gridDim.x) * RG);
  const int steps = (a.k + 32 * V - 1) / (32 * V);
  const int s0 = (int)((long long)steps * ks / a.k_split), s1 = (int)((long long)steps * (ks + 1) / a.k_split);
  const TW* w = reinterpret_cast<const TW*>(a.w);
  const TX* x = reinterpret_cast<const TX*>(a.x);
  pdl_wait();
  pdl_trigger();
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
          if (GATE) v = few_act<sizeof(TW) == 2>(a.act, v) * u;
          reinterpret_cast<TO*>(a.out)[(long long)m * a.ldo + col + j] = from_f<TO>(v);
        }
      }
    }
  }
}

// The second product is launched as a programmatic dependent of the first (1 token, 2048 x 8192 bf16: 23.2 -> 21.9 us;
// with its weights prefetched into L2 before its wait 22.6).
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
  return (int)launch_k_if((!GATE && pdl_in_call()) || pdl_enabled(), ffn_few_kernel<TW, TX, TO, MT, V, GATE>, dim3(grid), dim3(FEW_THREADS), 0, st, a);
}
// ---- more tokens: the warps' matrix instruction ------------------------------------------------------------------------
// A block multiplies 32 tokens (8 NT) with 32 weight rows (gate: 16 gate rows and their up rows, which meet in one thread); its
// four warps, and the blocks of a cluster, share the steps of 32 k.  A lane takes eight consecutive k of a weight row or a token
// straight from global memory: the order of k inside a step is free as long as both factors have the same one, so no operand
// passes through shared memory, and the next step's loads are under way while this one's are multiplied.  fp32 factors are split
// into three bf16 parts in registers (six products, the small ones first) and the instruction's sum, which is truncated, is added
// to the fp32 one after every step.  The warps' sums, then those of the cluster, are added in a fixed order.  Bound by the
// latency of a step (loads, splitting, 96 matrix instructions; eight warps per SM by their registers): 32 tokens fp32, 650 x
// 2600, 26 us for 20 MB of weights (the same tile on the fp32 units, fed through shared memory: 31; 2048 x 8192: 125, here 93).
#define FM_WARPS 4
#define FM_MI 2                      // instructions' rows of a warp: 2 x 16 (one: 2048 x 8192 fp32, 16 tokens 97 us, two 79)
#define FM_ROWS (16 * FM_MI)
#define FM_LD 33                     // floats per row of sums

// a lane's eight elements; left: elements from p to the end of the row, zeros behind it
template <typename TX, int V>
__device__ __forceinline__ void fm_load(const TX* p, int left, uint32_t (&r)[8 * sizeof(TX) / 4]) {
  constexpr int B = V * (int)sizeof(TX);
#pragma unroll
  for (int q = 0; q < 8 / V; ++q) {
    const bool in = q * V < left;
    if constexpr (B == 16) {
      const uint4 u = in ? *reinterpret_cast<const uint4*>(p + q * V) : make_uint4(0, 0, 0, 0);
      r[4 * q] = u.x; r[4 * q + 1] = u.y; r[4 * q + 2] = u.z; r[4 * q + 3] = u.w;
    } else if constexpr (B == 8) {
      const uint2 u = in ? *reinterpret_cast<const uint2*>(p + q * V) : make_uint2(0, 0);
      r[2 * q] = u.x; r[2 * q + 1] = u.y;
    } else if constexpr (B == 4) {
      r[q] = in ? *reinterpret_cast<const uint32_t*>(p + q * V) : 0u;
    } else {
      const uint32_t u = in ? *reinterpret_cast<const unsigned short*>(p + q) : 0u;
      if (q & 1) r[q / 2] |= u << 16;
      else r[q / 2] = u;
    }
  }
}
// the four registers of the instruction, for each part
template <typename T, typename TX, int S>
__device__ __forceinline__ void fm_parts(const uint32_t (&r)[8 * sizeof(TX) / 4], uint32_t (&q)[S][4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (sizeof(TX) == 2) {
      q[0][e] = r[e];
    } else if constexpr (S == 1) {
      Vec<T, 2> v;
      v.e[0] = from_f<T>(__uint_as_float(r[2 * e]));
      v.e[1] = from_f<T>(__uint_as_float(r[2 * e + 1]));
      q[0][e] = *reinterpret_cast<const uint32_t*>(v.e);
    } else {
      uint32_t w[3];
      split3(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]), w);
#pragma unroll
      for (int s = 0; s < 3; ++s) q[s][e] = w[s];
    }
  }
}
// c += A B over sixteen k; a0, a2: row lane / 4, a1, a3: row lane / 4 + 8; c: columns 2 (lane % 4) + 0, 1 of those rows
template <bool HALF>
__device__ __forceinline__ void fm_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (HALF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// blocks that an SM holds by their registers (fp32, 32 tokens, three with the tokens' loads one instruction ahead only: 31 against
// 26 us, 2048 x 8192 141 against 93)
template <typename TW, int NT>
constexpr int fm_resident() { return sizeof(TW) == 4 && NT == 4 ? 2 : 3; }

template <typename TW, typename TX, typename TO, int NT, int V, bool GATE>
__global__ void __launch_bounds__(32 * FM_WARPS, (fm_resident<TW, NT>())) ffn_mma_kernel(FewArgs a) {
  constexpr int S = sizeof(TW) == 4 ? 3 : 1, VX = V * (int)sizeof(TX) > 16 ? 16 / (int)sizeof(TX) : V;
  constexpr bool HALF = std::is_same<TW, __half>::value;
  __shared__ float sums[FM_WARPS * FM_ROWS * FM_LD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, k0 = 8 * (lane & 3);
  const int slices = a.k_split;              // blocks of a cluster
  const int slice = (int)(blockIdx.x % slices), c0 = (int)(blockIdx.x / slices) * (GATE ? FM_ROWS / 2 : FM_ROWS), m0 = (int)blockIdx.y * 32;
  const int steps = (a.k + 31) / 32, part = slice * FM_WARPS + warp, parts = slices * FM_WARPS;
  const int s0 = (int)((long long)steps * part / parts), s1 = (int)((long long)steps * (part + 1) / parts);
  const TW* w[FM_MI][2];
  const TX* x[NT];
#pragma unroll
  for (int i = 0; i < FM_MI; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {            // past the last column or token: that one again, not stored
      const int c = min(c0 + (GATE ? 8 * i : 16 * i + 8 * h) + g, a.n - 1);
      w[i][h] = reinterpret_cast<const TW*>(a.w) + (long long)c * a.ldw + (GATE && h ? a.up : 0) + k0;
    }
#pragma unroll
  for (int j = 0; j < NT; ++j) x[j] = reinterpret_cast<const TX*>(a.x) + (long long)min(m0 + 8 * j + g, a.m - 1) * a.ldx + k0;
  uint32_t rw[FM_MI][2][8 * sizeof(TW) / 4], rx[NT][8 * sizeof(TX) / 4];
  const auto load_w = [&](int s) {
#pragma unroll
    for (int i = 0; i < FM_MI; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) fm_load<TW, V>(w[i][h] + s * 32, a.k - s * 32 - k0, rw[i][h]);
  };
  pdl_wait();
  pdl_trigger();
  if (s0 < s1) {
    load_w(s0);
#pragma unroll
    for (int j = 0; j < NT; ++j) fm_load<TX, VX>(x[j] + s0 * 32, a.k - s0 * 32 - k0, rx[j]);
  }
  float acc[FM_MI][NT][4] = {};
#pragma unroll 1
  for (int s = s0; s < s1; ++s) {
    uint32_t p[FM_MI][2][S][4];
#pragma unroll
    for (int i = 0; i < FM_MI; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) fm_parts<TW, TW, S>(rw[i][h], p[i][h]);
    if (s + 1 < s1) load_w(s + 1);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      uint32_t q[S][4];
      fm_parts<TW, TX, S>(rx[j], q);
      if (s + 1 < s1) fm_load<TX, VX>(x[j] + (s + 1) * 32, a.k - (s + 1) * 32 - k0, rx[j]);
      float c[FM_MI][2][4] = {};             // a sum for each half of the step: more independent instructions
#pragma unroll
      for (int o = S - 1; o >= 0; --o)       // parts u of the weight and o - u of the token
#pragma unroll
        for (int u = 0; u <= o; ++u)
#pragma unroll
          for (int e = 0; e < 4; e += 2)
#pragma unroll
            for (int i = 0; i < FM_MI; ++i)
              fm_mma<HALF>(c[i][e / 2], p[i][0][u][e], p[i][1][u][e], p[i][0][u][e + 1], p[i][1][u][e + 1], q[o - u][e], q[o - u][e + 1]);
#pragma unroll
      for (int i = 0; i < FM_MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] += c[i][0][e] + c[i][1][e];
    }
  }
  // sums [warp][row][token]; gate: rows 0 .. 15 the gate's, 16 .. 31 the up rows'
#pragma unroll
  for (int i = 0; i < FM_MI; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = GATE ? FM_ROWS / 2 * (e >> 1) + 8 * i + g : 16 * i + 8 * (e >> 1) + g;
        sums[(warp * FM_ROWS + r) * FM_LD + 8 * j + 2 * (lane & 3) + (e & 1)] = acc[i][j][e];
      }
  __syncthreads();
  for (int i = threadIdx.x; i < FM_ROWS * 8 * NT; i += 32 * FM_WARPS) {
    const int at = i / (8 * NT) * FM_LD + i % (8 * NT);
    float v = sums[at];
#pragma unroll
    for (int q = 1; q < FM_WARPS; ++q) v += sums[q * FM_ROWS * FM_LD + at];
    sums[at] = v;
  }
  if (slices > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else __syncthreads();
  const uint32_t mine = (uint32_t)__cvta_generic_to_shared(sums);
  // of a cluster, every block writes its share of the results; consecutive threads take consecutive columns of a token
  constexpr int COLS = GATE ? FM_ROWS / 2 : FM_ROWS, OUT = COLS * 8 * NT;
  for (int i = slice * 32 * FM_WARPS + threadIdx.x; i < OUT; i += slices * 32 * FM_WARPS) {
    const int r = i % COLS, m = i / COLS;
    float v = 0.f, u = 0.f;
    for (int q = 0; q < slices; ++q) {
      float y, z = 0.f;
      uint32_t at;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(mine), "r"(q));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(y) : "r"(at + (r * FM_LD + m) * 4) : "memory");
      if (GATE) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(z) : "r"(at + ((r + FM_ROWS / 2) * FM_LD + m) * 4) : "memory");
      v += y;
      u += z;
    }
    if (c0 + r < a.n && m0 + m < a.m) {
      if (GATE) v = few_act<sizeof(TW) == 2>(a.act, v) * u;
      reinterpret_cast<TO*>(a.out)[(long long)(m0 + m) * a.ldo + c0 + r] = from_f<TO>(v);
    }
  }
  // the other blocks have read this one's sums
  if (slices > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename TW, typename TX, typename TO, int NT, int V, bool GATE>
static int fm_launch(FewArgs& a, cudaStream_t st) {
  const int tiles = (a.n + (GATE ? FM_ROWS / 2 : FM_ROWS) - 1) / (GATE ? FM_ROWS / 2 : FM_ROWS), groups = (a.m + 31) / 32, steps = (a.k + 31) / 32;
  a.k_split = 1;
  // blocks that share k: the cheapest by  rounds x (steps of a warp x cost of a step, which grows by a quarter with every further
  // block on the SM + what a block costs besides, about three steps)
  const int resident = fm_resident<TW, NT>();
  long long best = 1LL << 62;
  for (int q = 1; q <= 8 && (q - 1) * FM_WARPS < steps; q *= 2) {
    const long long blocks = (long long)tiles * groups * q, each = (blocks + sm_count() - 1) / sm_count();
    const long long rounds = (each + resident - 1) / resident, step = 3 + (each < resident ? each : resident);
    const long long cost = rounds * ((steps + q * FM_WARPS - 1) / (q * FM_WARPS) * step + 12);
    if (cost < best) { best = cost; a.k_split = q; }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * a.k_split), (unsigned)groups);
  cfg.blockDim = dim3(32 * FM_WARPS);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (a.k_split > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = a.k_split;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if ((!GATE && pdl_in_call()) || pdl_enabled()) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return (int)cudaLaunchKernelEx(&cfg, ffn_mma_kernel<TW, TX, TO, NT, V, GATE>, a);
}

template <typename TW, typename TX, typename TO, int V, bool GATE>
static int few_tokens(FewArgs& a, cudaStream_t st) {
  if (a.m <= 1) return few_launch<TW, TX, TO, 1, V, GATE>(a, st);
  if (a.m <= 2) return few_launch<TW, TX, TO, 2, V, GATE>(a, st);
  if (a.m <= 4) return few_launch<TW, TX, TO, 4, V, GATE>(a, st);
  if constexpr (sizeof(TW) == 4) {
    if (a.m <= 8) return few_launch<TW, TX, TO, 8, V, GATE>(a, st);
  } else {
    if (a.m <= 8) return fm_launch<TW, TX, TO, 1, V, GATE>(a, st);
  }
  if (a.m <= 16) return fm_launch<TW, TX, TO, 2, V, GATE>(a, st);
  return fm_launch<TW, TX, TO, 4, V, GATE>(a, st);
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

bool ffn_few_fits(int m, int d, int f, int n, int dt) {
  if (dt == DT_F32) return m <= 32;
  return m <= 4 || (m <= 16 && 2LL * f * d + (long long)n * f <= (1LL << 25));
}

int ffn_few_forward(const void* x, long long ldx, const void* w_in, long long ld_in, const void* w_out, long long ld_out, float* h,
                    void* y, int m, int d, int f, int n, int act, int dt, cudaStream_t st) {
  if (!ffn_few_fits(m, d, f, n, dt)) return -1;
  const long long ldh = (f + 15) / 16 * 16;
  FewArgs in = {w_in, x, h, ld_in, (long long)f * ld_in, ldx, ldh, m, f, d, act, 1};
  FewArgs out = {w_out, h, y, ld_out, 0, ldh, n, m, n, f, act, 1};
  if (dt == DT_F32) return few_forward<float>(in, out, st);
  if (dt == DT_BF16) return few_forward<__nv_bfloat16>(in, out, st);
  return few_forward<__half>(in, out, st);
}
