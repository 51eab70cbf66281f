// Gated feed-forward block on the 5th-generation tensor cores, forward and backward.
//
//   [G | U] = X W_in^T     W_in [2 F, D], gate rows first        H = act(G) * U            Y = H W_out^T      W_out [N, F]
//   dH = dY W_out          dG = dH U act'(G),  dU = dH act(G)    dX = dG W_in[:F] + dU W_in[F:]
//   dW_in = [dG | dU]^T X                                        dW_out = dY^T H
//
// Six products of one kernel (ffn_gemm_kernel), which differ in the operands' orientation and in the epilogue:
//   gate    both projections of a tile in ONE accumulator (the B tile holds BN / 2 gate rows and the BN / 2 up rows
//           that belong to them); the epilogue applies activation and product, so G and U meet in registers
//   dgate   dH stays in the accumulator: the epilogue reads G and U and writes dG and dU
//   plain   the four others
// No operand is ever transposed in memory: a tile is fetched K-major or MN-major, whichever way the tensor lies.
//
// Pipeline: one TMA thread, one thread that issues tcgen05.mma (kind::f16, M = 128, fp32 accumulators in TMEM), four
// epilogue warps; operands in a ring of 128-byte-swizzled stages of 64 k, accumulators double-buffered so that the
// epilogue of a tile runs under the multiplications of the next (persistent CTAs).
//
// Precision.  bf16 / fp16: operands as they are, fp32 accumulators; H and [dG | dU] are rounded once to the operands' type,
// because the next product reads them as tensor-core operands; G and U are kept in fp32 for the backward pass.
// fp32: every operand is the sum of three bf16 numbers (x = x1 + x2 + x3, each the rounded remainder of the ones before:
// 24 significant bits), a product is a1 b1 + (a1 b2 + a2 b1) + (a1 b3 + a2 b2 + a3 b1), what is left out is below 2^-24 of
// it.  The tensor core truncates when it adds to its accumulator, which over a long K costs far more than that
// (measured, one pass of exactly representable operands: relative error 7e-8 at K = 64, 4.4e-6 at K = 2600), so the fp32
// form takes its accumulator out after every 64 k and adds it up in registers; within those the small products go first.
//
// Every mbarrier wait is bounded; a wait that runs out sets the error word, the CTA drains and frees its TMEM.
#include "launch.cuh"
#include "tc_common.cuh"
#include "vec.cuh"

#define FF_BM 128
#define FF_BK 64             // k per stage: 128 bytes of 16-bit operands = one swizzle row
#define FF_THREADS 192       // warps 0-3 epilogue (warp 0 owns TMEM), warp 4 TMA, warp 5 MMA

#define FF_GATE 0
#define FF_DGATE 1
#define FF_PLAIN 2

#define ACT_SILU 0
#define ACT_GELU 1
#define ACT_RELU 2
#define ACT_SIGMOID 3

__device__ int g_ffn_error;

struct FfnGemm {
  CUtensorMap a, b;
  int M, N;              // output rows (of one part) and columns; gate: N = F
  int k_blocks;          // 64-wide k-blocks of one segment
  int segments;          // dX: 2 (gate and up rows of W_in); else 1
  int m_parts;           // dW_in: 2 (dG and dU); else 1
  int a_parts, b_parts;  // planes per split of the operand (2: gate / up)
  int a_mn, b_mn;        // operand lies MN-major
  int fp16;              // operand type: fp16 instead of bf16 (S = 1)
  int act;
  void* out;             // plain: [m_parts M, N];  gate: H [S][M][ldo];  dgate: dZ [S][2][M][ldo]
  int out_dt;            // plain: type of out
  int vec_ok;            // out's rows start on 16-byte boundaries
  long long ldo;
  float* z;              // gate: written (null in evaluation);  dgate: read;  [2][M][ldz]
  long long ldz;
};

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void umma_f16(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(acc) : "memory");
}
// 32 columns of this warp's 32 lanes; the caller waits
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ bool ff_epi_bar_or(bool flag) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, 1, 128, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r) : "r"((uint32_t)flag) : "memory");
  return r != 0;
}

// x as three bf16 numbers (finite x whose rounding would overflow is cut instead; the remainders of a non-finite x are zero)
__device__ __forceinline__ void split3(float x, __nv_bfloat16 (&p)[3]) {
  p[0] = __float2bfloat16_rn(x);
  if (!isfinite(__bfloat162float(p[0]))) p[0] = __float2bfloat16_rz(x);
  float r = x - __bfloat162float(p[0]);
  if (!isfinite(r)) r = 0.f;
  p[1] = __float2bfloat16_rn(r);
  p[2] = __float2bfloat16_rn(r - __bfloat162float(p[1]));
}

// activation and (wanted) its derivative
template <bool GRAD>
__device__ __forceinline__ float ff_act(int act, float z, float& slope) {
  if (act == ACT_GELU) {
    const float cdf = 0.5f * (1.f + erff(z * 0.70710678118654752f));
    if (GRAD) slope = fmaf(z * 0.39894228040143268f, expf(-0.5f * z * z), cdf);
    return z * cdf;
  }
  if (act == ACT_RELU) {
    if (GRAD) slope = z > 0.f ? 1.f : 0.f;
    return z < 0.f ? 0.f : z;
  }
  const float sg = 1.f / (1.f + expf(-z));
  if (act == ACT_SILU) {
    if (GRAD) slope = sg * fmaf(z, 1.f - sg, 1.f);
    return z * sg;
  }
  if (GRAD) slope = sg * (1.f - sg);
  return sg;
}

// eight consecutive values of one row into a 16-bit operand buffer (S planes); rows are padded to multiples of eight
template <int S>
__device__ __forceinline__ void ff_store_operand(void* base, long long plane, long long off, int fp16, const float* v) {
  if (S == 3) {
    Vec<__nv_bfloat16, 8> q[3];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      __nv_bfloat16 p[3];
      split3(v[e], p);
      q[0].e[e] = p[0]; q[1].e[e] = p[1]; q[2].e[e] = p[2];
    }
#pragma unroll
    for (int s = 0; s < 3; ++s) q[s].store(reinterpret_cast<__nv_bfloat16*>(base) + s * plane + off);
  } else if (fp16) {
    Vec<__half, 8> q;
#pragma unroll
    for (int e = 0; e < 8; ++e) q.e[e] = __float2half_rn(v[e]);
    q.store(reinterpret_cast<__half*>(base) + off);
  } else {
    Vec<__nv_bfloat16, 8> q;
#pragma unroll
    for (int e = 0; e < 8; ++e) q.e[e] = __float2bfloat16_rn(v[e]);
    q.store(reinterpret_cast<__nv_bfloat16*>(base) + off);
  }
}
template <typename T>
__device__ __forceinline__ void ff_store_plain(T* out, int n, bool vec, const float* v) {
  if (vec && n >= 8) {
    if (sizeof(T) == 4) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        Vec<T, 16 / sizeof(T)> q;
#pragma unroll
        for (int e = 0; e < 16 / (int)sizeof(T); ++e) q.e[e] = from_f<T>(v[(4 * h + e) & 7]);
        q.store(out + 4 * h);
      }
    } else {
      Vec<T, 16 / sizeof(T)> q;
#pragma unroll
      for (int e = 0; e < 16 / (int)sizeof(T); ++e) q.e[e] = from_f<T>(v[e]);
      q.store(out);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) out[e] = from_f<T>(v[e]);
  }
}

// the epilogue of columns [col, col + 8) of one row: v = accumulator (gate: G in v, U in u)
template <int S, int KIND>
__device__ __forceinline__ void ff_epilogue8(const FfnGemm& g, int m_part, int row, int col, const float* v, const float* u) {
  if (KIND == FF_GATE) {
    float h[8], slope;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = ff_act<false>(g.act, v[e], slope) * u[e];
    ff_store_operand<S>(g.out, (long long)g.M * g.ldo, (long long)row * g.ldo + col, g.fp16, h);
    if (g.z != nullptr) {
      float* z = g.z + (long long)row * g.ldz + col;
      *reinterpret_cast<float4*>(z) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(z + 4) = make_float4(v[4], v[5], v[6], v[7]);
      z += (long long)g.M * g.ldz;
      *reinterpret_cast<float4*>(z) = make_float4(u[0], u[1], u[2], u[3]);
      *reinterpret_cast<float4*>(z + 4) = make_float4(u[4], u[5], u[6], u[7]);
    }
  } else if (KIND == FF_DGATE) {
    const float* z = g.z + (long long)row * g.ldz + col;
    float zg[8], zu[8], dg[8], du[8];
    *reinterpret_cast<float4*>(zg) = *reinterpret_cast<const float4*>(z);
    *reinterpret_cast<float4*>(zg + 4) = *reinterpret_cast<const float4*>(z + 4);
    z += (long long)g.M * g.ldz;
    *reinterpret_cast<float4*>(zu) = *reinterpret_cast<const float4*>(z);
    *reinterpret_cast<float4*>(zu + 4) = *reinterpret_cast<const float4*>(z + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float slope;
      const float a = ff_act<true>(g.act, zg[e], slope);
      du[e] = v[e] * a;
      dg[e] = v[e] * zu[e] * slope;
    }
    const long long plane = (long long)g.M * g.ldo, off = (long long)row * g.ldo + col;
    ff_store_operand<S>(g.out, 2 * plane, off, g.fp16, dg);
    ff_store_operand<S>(g.out, 2 * plane, plane + off, g.fp16, du);
  } else {
    const long long off = ((long long)m_part * g.M + row) * g.ldo + col;
    const int n = g.N - col;
    if (g.out_dt == DT_F32) ff_store_plain(reinterpret_cast<float*>(g.out) + off, n, g.vec_ok, v);
    else if (g.out_dt == DT_BF16) ff_store_plain(reinterpret_cast<__nv_bfloat16*>(g.out) + off, n, g.vec_ok, v);
    else ff_store_plain(reinterpret_cast<__half*>(g.out) + off, n, g.vec_ok, v);
  }
}

template <int BN, int S> struct FfnSmem {
  static constexpr int A_TILE = FF_BM * FF_BK * 2, B_TILE = BN * FF_BK * 2;
  static constexpr int STAGE = S * (A_TILE + B_TILE);
  static constexpr int STAGES = (216 * 1024) / STAGE > 8 ? 8 : (216 * 1024) / STAGE;
  static constexpr int BYTES = STAGES * STAGE + 256 + 1024;
};

template <int BN, int S, int KIND>
__global__ void __launch_bounds__(FF_THREADS, 1) ffn_gemm_kernel(const __grid_constant__ FfnGemm g) {
  typedef FfnSmem<BN, S> L;
  extern __shared__ uint8_t smem_raw[];
  // 1024-byte alignment: the swizzle pattern is a function of the shared-memory address bits
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::STAGES * L::STAGE);
  uint64_t* empty = full + L::STAGES;
  uint64_t* acc_full = empty + L::STAGES;    // [2]
  uint64_t* acc_empty = acc_full + 2;        // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  constexpr int BN_OUT = KIND == FF_GATE ? BN / 2 : BN;    // output columns of a tile

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles_m = (g.M + FF_BM - 1) / FF_BM, tiles_n = (g.N + BN_OUT - 1) / BN_OUT;
  const int n_tiles = tiles_m * g.m_parts * tiles_n;
  const int n_kb = g.k_blocks * g.segments;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full + b, 1);
      mbar_init(acc_empty + b, 4);   // one arrival per epilogue warp
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  constexpr uint32_t TMEM_COLS = 2 * BN;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  if (warp == 4 && lane == 0) {
    // ---------------- TMA producer ----------------
    uint32_t it = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x) {
      const int tm = tile % (tiles_m * g.m_parts), n0 = (tile / (tiles_m * g.m_parts)) * BN_OUT;
      const int m_part = tm / tiles_m, m0 = (tm % tiles_m) * FF_BM;
      for (int i = 0; i < n_kb; ++i, ++it) {
        const uint32_t s = it % L::STAGES;
        if (it >= L::STAGES && !mbar_wait(empty + s, ((it / L::STAGES) - 1) & 1)) ok = false;
        if (*abort_flag) ok = false;
        if (!ok) { *abort_flag = 1; break; }
        const int seg = i / g.k_blocks, k0 = (i - seg * g.k_blocks) * FF_BK;
        mbar_expect_tx(full + s, L::STAGE);
        uint8_t* stage = smem + s * L::STAGE;
#pragma unroll
        for (int q = 0; q < S; ++q) {
          uint8_t* dA = stage + q * L::A_TILE;
          uint8_t* dB = stage + S * L::A_TILE + q * L::B_TILE;
          const int pa = q * g.a_parts + (g.m_parts > 1 ? m_part : (g.a_parts > 1 ? seg : 0));
          if (!g.a_mn) {
            tma_load_3d(dA, &g.a, full + s, k0, m0, pa);
          } else {
#pragma unroll
            for (int j = 0; j < FF_BM / 64; ++j) tma_load_3d(dA + j * 8192, &g.a, full + s, m0 + 64 * j, k0, pa);
          }
          if (KIND == FF_GATE) {
            tma_load_3d(dB, &g.b, full + s, k0, n0, q * 2);
            tma_load_3d(dB + L::B_TILE / 2, &g.b, full + s, k0, n0, q * 2 + 1);
          } else {
            const int pb = q * g.b_parts + (g.b_parts > 1 ? seg : 0);
            if (!g.b_mn) {
              tma_load_3d(dB, &g.b, full + s, k0, n0, pb);
            } else {
#pragma unroll
              for (int j = 0; j < BN / 64; ++j) tma_load_3d(dB + j * 8192, &g.b, full + s, n0 + 64 * j, k0, pb);
            }
          }
        }
      }
    }
  } else if (warp == 5 && lane == 0) {
    // ---------------- MMA issuer ----------------
    // instruction descriptor: fp32 accumulate, operand type, majorness bits, N >> 3, M >> 4
    const uint32_t type = g.fp16 ? 0u : 1u;
    const uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)g.a_mn << 15) | ((uint32_t)g.b_mn << 16) |
                           ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(FF_BM >> 4) << 24);
    // K-major: 16 k = 32 bytes further inside the 128-byte row, 8-row groups 1024 bytes apart; MN-major: 16 k = 16 rows of
    // 128 bytes, 8-k groups 1024 bytes apart, blocks of 64 MN elements 8192 bytes apart
    const uint32_t a_step = g.a_mn ? 2048 : 32, b_step = g.b_mn ? 2048 : 32;
    const uint32_t a_lbo = g.a_mn ? 8192 : 16, b_lbo = g.b_mn ? 8192 : 16;
    uint32_t it = 0, chunk = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < n_tiles && ok; tile += gridDim.x) {
      for (int i = 0; i < n_kb; ++i, ++it) {
        const bool first = S == 3 || i == 0;
        const uint32_t buf = chunk & 1;
        if (first && chunk >= 2 && !mbar_wait(acc_empty + buf, ((chunk >> 1) - 1) & 1)) ok = false;
        const uint32_t s = it % L::STAGES;
        if (ok && !mbar_wait(full + s, (it / L::STAGES) & 1)) ok = false;
        if (!ok) { *abort_flag = 1; break; }
        tc_fence_after();
        const uint32_t d = tmem_base + buf * BN;
        const uint32_t a_addr = smem_u32(smem + s * L::STAGE), b_addr = a_addr + S * L::A_TILE;
        if (S == 1) {
#pragma unroll
          for (int k = 0; k < FF_BK / 16; ++k)
            umma_f16(d, make_desc(a_addr + k * a_step, a_lbo, 1024), make_desc(b_addr + k * b_step, b_lbo, 1024), idesc,
                     (i > 0 || k > 0) ? 1u : 0u);
        } else {
          // smallest products first: (1,3) (3,1) (2,2) (1,2) (2,1) (1,1)
          constexpr int PA[6] = {0, 2, 1, 0, 1, 0}, PB[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
          for (int p = 0; p < 6; ++p)
#pragma unroll
            for (int k = 0; k < FF_BK / 16; ++k)
              umma_f16(d, make_desc(a_addr + PA[p] * L::A_TILE + k * a_step, a_lbo, 1024),
                       make_desc(b_addr + PB[p] * L::B_TILE + k * b_step, b_lbo, 1024), idesc, (p > 0 || k > 0) ? 1u : 0u);
        }
        tc_commit(empty + s);  // frees this stage once the MMAs above have read it
        if (S == 3 || i == n_kb - 1) {
          tc_commit(acc_full + buf);
          ++chunk;
        }
      }
    }
  } else if (warp < 4) {
    // ---------------- epilogue ----------------
    uint32_t chunk = 0;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    for (int tile = blockIdx.x; tile < n_tiles; tile += gridDim.x) {
      const int tm = tile % (tiles_m * g.m_parts), n0 = (tile / (tiles_m * g.m_parts)) * BN_OUT;
      const int m_part = tm / tiles_m, row = (tm % tiles_m) * FF_BM + warp * 32 + lane;
      bool stop = false;
      if (S == 3) {
        float acc[BN];
#pragma unroll
        for (int c = 0; c < BN; ++c) acc[c] = 0.f;
        for (int i = 0; i < n_kb; ++i, ++chunk) {
          const uint32_t buf = chunk & 1;
          const bool bad = !mbar_wait(acc_full + buf, (chunk >> 1) & 1) || *abort_flag != 0;
          if (ff_epi_bar_or(bad)) { stop = true; break; }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < BN; c += 32) {
            float v[32];
            tmem_ld32(tmem_base + lanes + buf * BN + c, v);
#pragma unroll
            for (int e = 0; e < 32; ++e) acc[c + e] += v[e];
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty + buf);
        }
        if (!stop && row < g.M) {
#pragma unroll
          for (int c = 0; c < BN_OUT; c += 8)
            if (n0 + c < g.N) ff_epilogue8<S, KIND>(g, m_part, row, n0 + c, acc + c, acc + (KIND == FF_GATE ? BN / 2 + c : c));
        }
      } else {
        const uint32_t buf = chunk & 1;
        const bool bad = !mbar_wait(acc_full + buf, (chunk >> 1) & 1) || *abort_flag != 0;
        if (ff_epi_bar_or(bad)) stop = true;
        else {
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < BN_OUT; c += 32) {
            float v[32], u[32];
            tmem_ld32(tmem_base + lanes + buf * BN + c, v);
            if (KIND == FF_GATE) tmem_ld32(tmem_base + lanes + buf * BN + BN / 2 + c, u);
            if (row < g.M) {
#pragma unroll
              for (int e = 0; e < 32; e += 8)
                if (n0 + c + e < g.N) ff_epilogue8<S, KIND>(g, m_part, row, n0 + c + e, v + e, u + e);
            }
          }
          // the accumulator may be overwritten by the tile after next
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty + buf);
          ++chunk;
        }
      }
      if (stop) { *abort_flag = 1; break; }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) atomicExch(&g_ffn_error, 1);
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

// ---- operands: fp32 into three bf16 planes, 16-bit rows onto 16-byte boundaries -------------------------------------
// src [rows, cols] with lds elements per row -> dst [S][rows][ldd], ldd a multiple of eight; the tail columns are zero
template <typename T, int S>
__global__ void __launch_bounds__(256) ffn_operand_kernel(const T* src, long long rows, int cols, long long lds, void* dst, int ldd) {
  pdl_wait();
  pdl_trigger();
  const int per_row = ldd / 8;
  const long long total = rows * per_row;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long r = i / per_row;
    const int c = (int)(i - r * per_row) * 8;
    const T* p = src + r * lds + c;
    if (S == 3) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? to_f(p[e]) : 0.f;
      ff_store_operand<3>(dst, rows * ldd, r * ldd + c, 0, v);
    } else {
      Vec<T, 16 / sizeof(T)> q;
      q.clear();
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < cols) q.e[e] = p[e];
      q.store(reinterpret_cast<T*>(dst) + r * ldd + c);
    }
  }
}

// ---------------------------------- host side ----------------------------------------------
static inline int pad8(int n) { return (n + 7) / 8 * 8; }

// one 16-bit operand: S planes of `parts` matrices [rows, cols], `ld` elements per row
struct FfnOperand {
  const void* p;
  int rows, cols, parts, splits;
  long long ld;
};

static int ffn_map(CUtensorMap* map, const FfnOperand& o, int fp16, int mn_major, int box_rows) {
  TcEncodeTiledFn enc = tc_get_encode();
  if (enc == nullptr) return -10;
  if (((uintptr_t)o.p & 15) != 0 || o.ld % 8 != 0) return -11;
  cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)(o.parts * o.splits)};
  cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)o.ld * 2 * (cuuint64_t)o.rows};
  cuuint32_t box[3] = {64, (cuuint32_t)(mn_major ? FF_BK : box_rows), 1}, es[3] = {1, 1, 1};
  CUresult r = enc(map, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.p),
                   dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -12;
}

template <int BN, int S, int KIND>
static int ffn_launch_t(FfnGemm& g, const FfnOperand& a, const FfnOperand& b, cudaStream_t st) {
  constexpr int smem = FfnSmem<BN, S>::BYTES;
  // before the tensor maps: a runtime call makes the device's context current in a thread that has not used it yet
  // (autograd's), without which the driver refuses to encode a map
  cudaError_t e = cudaFuncSetAttribute(ffn_gemm_kernel<BN, S, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return (int)e;
  int rc = ffn_map(&g.a, a, g.fp16, g.a_mn, FF_BM);
  if (rc) return rc;
  rc = ffn_map(&g.b, b, g.fp16, g.b_mn, KIND == FF_GATE ? BN / 2 : BN);
  if (rc) return rc;
  const int bn_out = KIND == FF_GATE ? BN / 2 : BN;
  const long long tiles = (long long)((g.M + FF_BM - 1) / FF_BM) * g.m_parts * ((g.N + bn_out - 1) / bn_out);
  if (tiles > 0x7fffffffLL) return -1;
  const int grid = tiles < sm_count() ? (int)tiles : sm_count();
  return (int)launch_k(ffn_gemm_kernel<BN, S, KIND>, dim3(grid), dim3(FF_THREADS), (size_t)smem, st, g);
}

// Tile width by the number of tiles: the widest that still gives every SM one (a narrow tile reads more operand bytes per
// multiplication; an idle SM costs more).
template <int S, int KIND>
static int ffn_launch(FfnGemm& g, const FfnOperand& a, const FfnOperand& b, cudaStream_t st) {
  const long long m = (long long)((g.M + FF_BM - 1) / FF_BM) * g.m_parts;
  const int cols = KIND == FF_GATE ? 2 * g.N : g.N;
  if constexpr (S == 1) {
    if (m * ((cols + 255) / 256) >= sm_count()) return ffn_launch_t<256, S, KIND>(g, a, b, st);
  }
  if (m * ((cols + 127) / 128) >= sm_count()) return ffn_launch_t<128, S, KIND>(g, a, b, st);
  return ffn_launch_t<64, S, KIND>(g, a, b, st);
}
template <int KIND>
static int ffn_gemm(int splits, FfnGemm& g, const FfnOperand& a, const FfnOperand& b, cudaStream_t st) {
  return splits == 3 ? ffn_launch<3, KIND>(g, a, b, st) : ffn_launch<1, KIND>(g, a, b, st);
}

// A matrix the products can read: itself, or its image in the workspace (dst)
static int ffn_prepare(FfnOperand* o, const void* src, long long rows, int cols, long long ld, int parts, int dt, void* dst,
                       cudaStream_t st) {
  o->rows = (int)(rows / parts);
  o->cols = cols;
  o->parts = parts;
  o->splits = dt == DT_F32 ? 3 : 1;
  if (dst == nullptr) {
    o->p = src;
    o->ld = ld;
    return 0;
  }
  o->p = dst;
  o->ld = pad8(cols);
  if (src == nullptr) return 0;       // prepared by the forward pass
  const long long runs = rows * (pad8(cols) / 8);
  const long long blocks = (runs + 255) / 256, most = 16LL * sm_count();
  const dim3 grid((unsigned)(blocks < most ? blocks : most)), block(256);
  const int ldd = pad8(cols);
  if (dt == DT_F32)
    return (int)launch_k(ffn_operand_kernel<float, 3>, grid, block, 0, st, (const float*)src, rows, cols, ld, dst, ldd);
  return (int)launch_k(ffn_operand_kernel<uint16_t, 1>, grid, block, 0, st, (const uint16_t*)src, rows, cols, ld, dst, ldd);
}

struct FfnShape {
  int m, d, f, n, act, dt;
};
static bool ffn_shape_ok(const FfnShape& s) {
  const long long big = 0x7fffff00LL;
  return s.m > 0 && s.d > 0 && s.f > 0 && s.n > 0 && s.dt >= 0 && s.dt <= 2 && s.act >= 0 && s.act <= 3 &&
         s.m < big && s.d < big && 2LL * s.f < big && s.n < big;
}
static void ffn_out(FfnGemm& g, void* out, int dt, long long ldo) {
  g.out = out;
  g.out_dt = dt;
  g.ldo = ldo;
  g.vec_ok = ((uintptr_t)out & 15) == 0 && (ldo * dt_bytes(dt)) % 16 == 0;
}

// Every operand comes with an optional image: [S][rows][pad8(cols)] 16-bit elements, S = 3 for fp32, needed for fp32 and
// for rows that do not start on 16-byte boundaries.  h: [S][m][pad8(f)] 16-bit; z: [2][m][pad8(f)] fp32 or null.
extern "C" int gated_ffn_forward(const void* x, long long ldx, void* x_img, const void* w_in, long long ld_in, void* in_img,
                                 const void* w_out, long long ld_out, void* out_img, void* h, float* z, void* y, int m, int d,
                                 int f, int n, int act, int dt, cudaStream_t st) {
  const FfnShape s = {m, d, f, n, act, dt};
  if (!ffn_shape_ok(s)) return -1;
  FfnOperand ox, oi, oo;
  int rc = ffn_prepare(&ox, x, m, d, ldx, 1, dt, x_img, st);
  if (!rc) rc = ffn_prepare(&oi, w_in, 2LL * f, d, ld_in, 2, dt, in_img, st);
  if (!rc) rc = ffn_prepare(&oo, w_out, n, f, ld_out, 1, dt, out_img, st);
  if (rc) return rc;
  const int S = dt == DT_F32 ? 3 : 1;
  FfnGemm g = {};
  g.fp16 = dt == DT_F16;
  g.act = act;
  g.segments = g.m_parts = g.a_parts = 1;
  g.b_parts = 2;
  g.M = m; g.N = f; g.k_blocks = (d + FF_BK - 1) / FF_BK;
  g.out = h; g.ldo = pad8(f); g.z = z; g.ldz = pad8(f);
  rc = ffn_gemm<FF_GATE>(S, g, ox, oi, st);
  if (rc) return rc;
  const FfnOperand oh = {h, m, f, 1, S, pad8(f)};
  g.b_parts = 1;
  g.N = n; g.k_blocks = (f + FF_BK - 1) / FF_BK;
  ffn_out(g, y, dt, n);
  return ffn_gemm<FF_PLAIN>(S, g, oh, oo, st);
}

// x, w_in, w_out: as in the forward pass; where an image is given it holds the forward pass' image already.
// dz: [S][2][m][pad8(f)] 16-bit scratch.  dx, dw_in, dw_out may be null.
extern "C" int gated_ffn_backward(const void* x, long long ldx, void* x_img, const void* w_in, long long ld_in, void* in_img,
                                  const void* w_out, long long ld_out, void* out_img, const void* dy, long long ldy,
                                  void* dy_img, const void* h, const float* z, void* dz, void* dx, void* dw_in, void* dw_out,
                                  int m, int d, int f, int n, int act, int dt, cudaStream_t st) {
  const FfnShape s = {m, d, f, n, act, dt};
  if (!ffn_shape_ok(s)) return -1;
  const int S = dt == DT_F32 ? 3 : 1;
  FfnOperand ox, oi, oo, oy;
  int rc = ffn_prepare(&oy, dy, m, n, ldy, 1, dt, dy_img, st);
  if (!rc) rc = ffn_prepare(&ox, x_img != nullptr ? nullptr : x, m, d, ldx, 1, dt, x_img, st);
  if (!rc) rc = ffn_prepare(&oi, in_img != nullptr ? nullptr : w_in, 2LL * f, d, ld_in, 2, dt, in_img, st);
  if (!rc) rc = ffn_prepare(&oo, out_img != nullptr ? nullptr : w_out, n, f, ld_out, 1, dt, out_img, st);
  if (rc) return rc;
  const FfnOperand oh = {h, m, f, 1, S, pad8(f)}, oz = {dz, m, f, 2, S, pad8(f)};
  FfnGemm base = {};
  base.fp16 = dt == DT_F16;
  base.act = act;
  base.segments = base.m_parts = base.a_parts = base.b_parts = 1;
  FfnGemm g = base;
  if (dx != nullptr || dw_in != nullptr) {
    g.M = m; g.N = f; g.k_blocks = (n + FF_BK - 1) / FF_BK; g.b_mn = 1;
    g.out = dz; g.ldo = pad8(f); g.z = const_cast<float*>(z); g.ldz = pad8(f);
    if ((rc = ffn_gemm<FF_DGATE>(S, g, oy, oo, st))) return rc;
  }
  if (dx != nullptr) {
    g = base;
    g.M = m; g.N = d; g.k_blocks = (f + FF_BK - 1) / FF_BK; g.segments = 2; g.a_parts = g.b_parts = 2; g.b_mn = 1;
    ffn_out(g, dx, dt, d);
    if ((rc = ffn_gemm<FF_PLAIN>(S, g, oz, oi, st))) return rc;
  }
  if (dw_in != nullptr) {
    g = base;
    g.M = f; g.N = d; g.k_blocks = (m + FF_BK - 1) / FF_BK; g.m_parts = g.a_parts = 2; g.a_mn = g.b_mn = 1;
    ffn_out(g, dw_in, dt, d);
    if ((rc = ffn_gemm<FF_PLAIN>(S, g, oz, ox, st))) return rc;
  }
  if (dw_out != nullptr) {
    g = base;
    g.M = n; g.N = f; g.k_blocks = (m + FF_BK - 1) / FF_BK; g.a_mn = g.b_mn = 1;
    ffn_out(g, dw_out, dt, f);
    if ((rc = ffn_gemm<FF_PLAIN>(S, g, oy, oh, st))) return rc;
  }
  return 0;
}

// 0, or 1 after a bounded wait of a kernel on the current device ran out (synchronises)
extern "C" int gated_ffn_last_error() {
  int v = -1;
  cudaMemcpyFromSymbol(&v, g_ffn_error, sizeof(int));
  return v;
}
