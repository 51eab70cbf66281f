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
// Pipeline: one TMA thread, one thread that issues tcgen05.mma (kind::f16, fp32 accumulators in TMEM), eight epilogue
// warps; operands in a ring of 128-byte-swizzled stages of 64 k, accumulators double-buffered so that the epilogue of a tile
// runs under the multiplications of the next (persistent CTAs).  Large products run as pairs of CTAs (cta_group::2, 256-row
// tiles): each CTA fetches half of the B tile, which halves its share of the operand traffic.
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

#define FF_BM 128            // accumulator rows of one CTA
#define FF_BK 64             // k per stage: 128 bytes of 16-bit operands = one swizzle row
#define FF_EPI 8             // epilogue warps 0-7 (warp 0 owns TMEM), warp 8 TMA, warp 9 MMA
#define FF_THREADS (32 * (FF_EPI + 2))

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
  int vec_bytes;         // plain: common alignment of out's rows (32, 16 or less)
  long long ldo;
  float* z;              // gate: written (null in evaluation);  dgate: read;  [2][M][ldz]
  long long ldz;
};

// ---- pairs of CTAs (cta_group::2) ----------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
// address of this CTA's shared-memory word in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t map_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// What these barriers hand over are operand tiles (complete_tx) and accumulators (tcgen05 fences and commits), no plain
// memory: the default scope serves.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// true in one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// CG = 2: the bytes are counted on a barrier of either CTA of the pair (`bar`: a cluster address)
template <int CG>
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  if (CG == 2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(smem_dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(smem_dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void umma_f16(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  if (CG == 2) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(acc) : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(acc) : "memory");
  }
}
// arrives on `bar` (CG = 2: of both CTAs) when the multiplications issued so far are done
template <int CG>
__device__ __forceinline__ void ff_commit(uint64_t* bar) {
  if (CG == 2) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
  } else {
    tc_commit(bar);
  }
}
template <int CG>
__device__ __forceinline__ void ff_tmem_alloc(uint32_t* slot, uint32_t cols) {
  if (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void ff_tmem_free(uint32_t base, uint32_t cols) {
  if (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
// 16 columns of this warp's 32 lanes; the caller waits (tmem_wait16) before it uses them
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// waits for all loads of this thread; the registers are operands, so that no use of them can move in front of it
__device__ __forceinline__ void tmem_wait16(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                 "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])::"memory");
}
__device__ __forceinline__ bool ff_epi_bar_or(bool flag) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, 1, %2, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r) : "r"((uint32_t)flag), "n"(FF_EPI * 32) : "memory");
  return r != 0;
}

// 32 bytes of a row with one access: a whole sector, although the lanes of a warp are in different rows
__device__ __forceinline__ void ld32b(const void* p, uint32_t* r) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "l"(p) : "memory");
}
__device__ __forceinline__ void st32b(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ uint32_t pack2(float a, float b, int fp16) {
  if (fp16) {
    const __half2 q = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&q);
  }
  const __nv_bfloat162 q = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&q);
}

// x as three bf16 numbers (finite x whose rounding would overflow is cut instead; the remainders of a non-finite x are zero)
__device__ __forceinline__ void split3(float x, float (&p)[3]) {
  p[0] = __bfloat162float(__float2bfloat16_rn(x));
  if (!isfinite(p[0])) p[0] = __bfloat162float(__float2bfloat16_rz(x));
  float r = x - p[0];
  if (!isfinite(r)) r = 0.f;
  p[1] = __bfloat162float(__float2bfloat16_rn(r));
  p[2] = r - p[1];
}

// activation and (wanted) its derivative; FAST: 16-bit results, for which the approximate exponential and quotient
// (relative error about 2^-21) are exact enough
template <bool GRAD, bool FAST>
__device__ __forceinline__ float ff_act(int act, float z, float& slope) {
  if (act == ACT_GELU) {
    const float cdf = 0.5f * (1.f + erff(z * 0.70710678118654752f));
    if (GRAD) {
      const float e = -0.5f * z * z;
      slope = fmaf(z * 0.39894228040143268f, FAST ? __expf(e) : expf(e), cdf);
    }
    return z * cdf;
  }
  if (act == ACT_RELU) {
    if (GRAD) slope = z > 0.f ? 1.f : 0.f;
    return z < 0.f ? 0.f : z;
  }
  // __fdividef gives 0 for divisors above 2^126, which is the limit wanted here
  const float sg = FAST ? __fdividef(1.f, 1.f + __expf(-z)) : 1.f / (1.f + expf(-z));
  if (act == ACT_SILU) {
    if (GRAD) slope = sg * fmaf(z, 1.f - sg, 1.f);
    return z * sg;
  }
  if (GRAD) slope = sg * (1.f - sg);
  return sg;
}

// sixteen consecutive values of one row into a 16-bit operand buffer (S planes); rows are padded to multiples of sixteen
template <int S>
__device__ __forceinline__ void ff_store_operand(uint16_t* base, long long plane, long long off, int fp16, const float* v) {
  if (S == 3) {
    uint32_t q[3][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float lo[3], hi[3];
      split3(v[2 * e], lo);
      split3(v[2 * e + 1], hi);
#pragma unroll
      for (int s = 0; s < 3; ++s) q[s][e] = pack2(lo[s], hi[s], 0);
    }
#pragma unroll
    for (int s = 0; s < 3; ++s) st32b(base + s * plane + off, q[s]);
  } else {
    uint32_t q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = pack2(v[2 * e], v[2 * e + 1], fp16);
    st32b(base + off, q);
  }
}
// n <= 16 of sixteen values to a row of the result; `bytes`: common alignment of its rows
template <typename T>
__device__ __forceinline__ void ff_store_plain(T* out, int n, int bytes, const float* v) {
  constexpr int W = 16 / (int)sizeof(T);
  if (n >= 16 && bytes >= 32) {
#pragma unroll
    for (int h = 0; h < 16; h += 2 * W) {
      union { T e[2 * W]; uint32_t r[8]; } q;
#pragma unroll
      for (int e = 0; e < 2 * W; ++e) q.e[e] = from_f<T>(v[h + e]);
      st32b(out + h, q.r);
    }
    return;
  }
  if (bytes >= 16) {
#pragma unroll
    for (int h = 0; h < 16; h += W) {
      if (h + W <= n) {
        Vec<T, W> q;
#pragma unroll
        for (int e = 0; e < W; ++e) q.e[e] = from_f<T>(v[h + e]);
        q.store(out + h);
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (h + e < n) out[h + e] = from_f<T>(v[h + e]);
      }
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (e < n) out[e] = from_f<T>(v[e]);
}

// The epilogue of columns [col, col + 16) of one row: v = accumulator (gate: G in v, U in u; dgate: G and U of the forward
// pass in zg, zu).  Buffers between the products have rows padded to sixteen elements: whole runs are written there.
template <int S, int KIND>
__device__ __forceinline__ void ff_epilogue16(const FfnGemm& g, int m_part, int row, int col, const float* v, const float* u,
                                              const float* zg, const float* zu) {
  constexpr bool FAST = S == 1;
  if (KIND == FF_GATE) {
    if (g.z != nullptr) {
      float* z = g.z + (long long)row * g.ldz + col;
      st32b(z, reinterpret_cast<const uint32_t*>(v));
      st32b(z + 8, reinterpret_cast<const uint32_t*>(v + 8));
      z += (long long)g.M * g.ldz;
      st32b(z, reinterpret_cast<const uint32_t*>(u));
      st32b(z + 8, reinterpret_cast<const uint32_t*>(u + 8));
    }
    float h[16], slope;
#pragma unroll
    for (int e = 0; e < 16; ++e) h[e] = ff_act<false, FAST>(g.act, v[e], slope) * u[e];
    ff_store_operand<S>(reinterpret_cast<uint16_t*>(g.out), (long long)g.M * g.ldo, (long long)row * g.ldo + col, g.fp16, h);
  } else if (KIND == FF_DGATE) {
    float dg[16], du[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float slope;
      const float a = ff_act<true, FAST>(g.act, zg[e], slope);
      du[e] = v[e] * a;
      dg[e] = v[e] * zu[e] * slope;
    }
    const long long plane = (long long)g.M * g.ldo, off = (long long)row * g.ldo + col;
    ff_store_operand<S>(reinterpret_cast<uint16_t*>(g.out), 2 * plane, off, g.fp16, dg);
    ff_store_operand<S>(reinterpret_cast<uint16_t*>(g.out), 2 * plane, plane + off, g.fp16, du);
  } else {
    const long long off = ((long long)m_part * g.M + row) * g.ldo + col;
    const int n = g.N - col;
    if (g.out_dt == DT_F32) ff_store_plain(reinterpret_cast<float*>(g.out) + off, n, g.vec_bytes, v);
    else if (g.out_dt == DT_BF16) ff_store_plain(reinterpret_cast<__nv_bfloat16*>(g.out) + off, n, g.vec_bytes, v);
    else ff_store_plain(reinterpret_cast<__half*>(g.out) + off, n, g.vec_bytes, v);
  }
}
// G and U of sixteen columns (dgate)
__device__ __forceinline__ void ff_load_z(const FfnGemm& g, int row, int col, float* zg, float* zu) {
  const float* z = g.z + (long long)row * g.ldz + col;
  ld32b(z, reinterpret_cast<uint32_t*>(zg));
  ld32b(z + 8, reinterpret_cast<uint32_t*>(zg + 8));
  z += (long long)g.M * g.ldz;
  ld32b(z, reinterpret_cast<uint32_t*>(zu));
  ld32b(z + 8, reinterpret_cast<uint32_t*>(zu + 8));
}

// BN accumulator columns, S operand planes, CG CTAs per tile: a pair (CG = 2) shares one 256-row tile, each CTA fetches its
// 128 rows of A and half of the B tile, so a byte of B serves 256 rows
template <int BN, int S, int CG> struct FfnSmem {
  static constexpr int A_TILE = FF_BM * FF_BK * 2, B_TILE = BN / CG * FF_BK * 2;
  static constexpr int STAGE = S * (A_TILE + B_TILE);
  static constexpr int STAGES = (216 * 1024) / STAGE > 8 ? 8 : (216 * 1024) / STAGE;
  static constexpr int BYTES = STAGES * STAGE + 256 + 1024;
};

// Tile order: groups of FF_GROUP row tiles, rows fastest within a group, so that the tiles worked on at one time form a
// block that is about as high as wide and share both operands' panels in L2.
#define FF_GROUP 8
__device__ __forceinline__ void ff_tile(int tile, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int per_group = FF_GROUP * tiles_n, group = tile / per_group, r = tile - group * per_group;
  const int rows = min(FF_GROUP, tiles_m - group * FF_GROUP);
  tn = r / rows;
  tm = group * FF_GROUP + (r - tn * rows);
}

template <int BN, int S, int KIND, int CG>
__global__ void __launch_bounds__(FF_THREADS, 1) ffn_gemm_kernel(const __grid_constant__ FfnGemm g) {
  typedef FfnSmem<BN, S, CG> L;
  extern __shared__ uint8_t smem_raw[];
  // 1024-byte alignment: the swizzle pattern is a function of the shared-memory address bits
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::STAGES * L::STAGE);   // CG = 2: the leader's count both CTAs' bytes
  uint64_t* empty = full + L::STAGES;
  uint64_t* acc_full = empty + L::STAGES;    // [2]
  uint64_t* acc_empty = acc_full + 2;        // [2], the leader's
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  constexpr int BN_OUT = KIND == FF_GATE ? BN / 2 : BN;    // output columns of a tile
  constexpr int TM = FF_BM * CG;                           // output rows of a tile

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  const int tiles_m = (g.M + TM - 1) / TM, tiles_n = (g.N + BN_OUT - 1) / BN_OUT;
  const int n_tiles = tiles_m * g.m_parts * tiles_n;
  const int n_kb = g.k_blocks * g.segments;
  const int first_tile = blockIdx.x / CG, tile_step = gridDim.x / CG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full + b, 1);
      mbar_init(acc_empty + b, FF_EPI * CG);   // one arrival per epilogue warp
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  constexpr uint32_t TMEM_COLS = 2 * BN;
  if (warp == 0) ff_tmem_alloc<CG>(tmem_slot, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_all();    // the peer's barriers exist
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  // The TMA and the MMA warp run their loops as whole warps and elect a lane for the instructions alone: addresses and
  // descriptors then stay in uniform registers.
  if (warp == FF_EPI) {
    // ---------------- TMA producer ----------------
    uint32_t it = 0, s = 0, phase = 1;      // stage and the parity of its `empty` barrier (the first round passes at once)
    bool ok = true;
    for (int tile = first_tile; tile < n_tiles && ok; tile += tile_step) {
      int tm, tn;
      ff_tile(tile, tiles_m * g.m_parts, tiles_n, tm, tn);
      const int n0 = tn * BN_OUT, m_part = tm / tiles_m, m0 = (tm % tiles_m) * TM + (int)rank * FF_BM;
      for (int seg = 0; seg < g.segments && ok; ++seg) {
        const int part_a = g.m_parts > 1 ? m_part : (g.a_parts > 1 ? seg : 0), part_b = g.b_parts > 1 ? seg : 0;
        for (int k0 = 0; k0 < g.k_blocks * FF_BK; k0 += FF_BK) {
          ok = __all_sync(0xffffffffu, mbar_wait(empty + s, phase) && *abort_flag == 0);
          if (!ok) break;
          if (elect_one()) {
            if (rank == 0) mbar_expect_tx(full + s, CG * L::STAGE);
            const uint32_t bar = CG == 2 ? map_rank(full + s, 0) : smem_u32(full + s);
            uint8_t* stage = smem + s * L::STAGE;
#pragma unroll
            for (int q = 0; q < S; ++q) {
              uint8_t* dA = stage + q * L::A_TILE;
              uint8_t* dB = stage + S * L::A_TILE + q * L::B_TILE;
              const int pa = q * g.a_parts + part_a;
              if (!g.a_mn) {
                tma_load_3d<CG>(dA, &g.a, bar, k0, m0, pa);
              } else {
#pragma unroll
                for (int j = 0; j < FF_BM / 64; ++j) tma_load_3d<CG>(dA + j * 8192, &g.a, bar, m0 + 64 * j, k0, pa);
              }
              if (KIND == FF_GATE) {
                // accumulator columns: BN / 2 gate, then BN / 2 up; of a pair, one CTA fetches the gate rows, the other the up rows
                if (CG == 2) {
                  tma_load_3d<CG>(dB, &g.b, bar, k0, n0, q * 2 + (int)rank);
                } else {
                  tma_load_3d<CG>(dB, &g.b, bar, k0, n0, q * 2);
                  tma_load_3d<CG>(dB + L::B_TILE / 2, &g.b, bar, k0, n0, q * 2 + 1);
                }
              } else {
                const int pb = q * g.b_parts + part_b, nb = n0 + (int)rank * (BN / CG);
                if (!g.b_mn) {
                  tma_load_3d<CG>(dB, &g.b, bar, k0, nb, pb);
                } else {
#pragma unroll
                  for (int j = 0; j < BN / CG / 64; ++j) tma_load_3d<CG>(dB + j * 8192, &g.b, bar, nb + 64 * j, k0, pb);
                }
              }
            }
          }
          __syncwarp();
          ++it;
          if (++s == L::STAGES) { s = 0; phase ^= 1; }
        }
      }
    }
    // after a wait that ran out: the copies in flight end before this CTA's shared memory is given back
    if (!ok) {
      *abort_flag = 1;
      if (rank == 0)
        for (uint32_t j = it > L::STAGES ? it - L::STAGES : 0; j < it; ++j) mbar_wait(full + j % L::STAGES, (j / L::STAGES) & 1);
    }
  } else if (warp == FF_EPI + 1 && rank == 0) {
    // ---------------- MMA issuer (of a pair: the leader's) ----------------
    // instruction descriptor: fp32 accumulate, operand type, majorness bits, N >> 3, M >> 4
    const uint32_t type = g.fp16 ? 0u : 1u;
    const uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)g.a_mn << 15) | ((uint32_t)g.b_mn << 16) |
                           ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
    // K-major: 16 k = 32 bytes further inside the 128-byte row, 8-row groups 1024 bytes apart; MN-major: 16 k = 16 rows of
    // 128 bytes, 8-k groups 1024 bytes apart, blocks of 64 MN elements 8192 bytes apart.  Descriptors count in 16 bytes.
    const uint32_t a_step = (g.a_mn ? 2048 : 32) >> 4, b_step = (g.b_mn ? 2048 : 32) >> 4;
    const uint32_t base = smem_u32(smem);
    const uint64_t da0 = make_desc(base, g.a_mn ? 8192 : 16, 1024), db0 = make_desc(base + S * L::A_TILE, g.b_mn ? 8192 : 16, 1024);
    uint32_t s = 0, phase = 0, chunk = 0;
    bool ok = true;
    for (int tile = first_tile; tile < n_tiles && ok; tile += tile_step) {
      for (int i = 0; i < n_kb; ++i) {
        const uint32_t buf = chunk & 1;
        // the first round of either accumulator passes at once
        if (S == 3 || i == 0) ok = mbar_wait(acc_empty + buf, ((chunk >> 1) & 1) ^ 1);
        ok = __all_sync(0xffffffffu, ok && mbar_wait(full + s, phase));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t d = tmem_base + buf * BN;
          const uint64_t da = da0 + s * (L::STAGE >> 4), db = db0 + s * (L::STAGE >> 4);
          if (S == 1) {
#pragma unroll
            for (int k = 0; k < FF_BK / 16; ++k) umma_f16<CG>(d, da + k * a_step, db + k * b_step, idesc, (i > 0 || k > 0) ? 1u : 0u);
          } else {
            // smallest products first: (1,3) (3,1) (2,2) (1,2) (2,1) (1,1)
            constexpr int PA[6] = {0, 2, 1, 0, 1, 0}, PB[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
            for (int p = 0; p < 6; ++p)
#pragma unroll
              for (int k = 0; k < FF_BK / 16; ++k)
                umma_f16<CG>(d, da + PA[p] * (L::A_TILE >> 4) + k * a_step, db + PB[p] * (L::B_TILE >> 4) + k * b_step, idesc,
                             (p > 0 || k > 0) ? 1u : 0u);
          }
          ff_commit<CG>(empty + s);  // frees this stage once the MMAs above have read it
          if (S == 3 || i == n_kb - 1) ff_commit<CG>(acc_full + buf);
        }
        __syncwarp();
        if (S == 3 || i == n_kb - 1) ++chunk;
        if (++s == L::STAGES) { s = 0; phase ^= 1; }
      }
    }
    if (!ok) *abort_flag = 1;
  } else if (warp < FF_EPI) {
    // ---------------- epilogue: warp w reads lanes 32 (w % 4) ... of half of the tile's output columns ----------------
    constexpr int HC = BN_OUT / 2;         // output columns per warp
    const int half = warp >> 2;
    uint32_t chunk = 0;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    for (int tile = first_tile; tile < n_tiles; tile += tile_step) {
      int tm, tn;
      ff_tile(tile, tiles_m * g.m_parts, tiles_n, tm, tn);
      const int n0 = tn * BN_OUT + half * HC, m_part = tm / tiles_m, row = (tm % tiles_m) * TM + (int)rank * FF_BM + (warp & 3) * 32 + lane;
      bool stop = false;
      if (S == 3) {
        // the accumulator of every 64 k, added up in registers
        constexpr int NA = KIND == FF_GATE ? 2 * HC : HC;
        float acc[NA];
#pragma unroll
        for (int c = 0; c < NA; ++c) acc[c] = 0.f;
        for (int i = 0; i < n_kb; ++i, ++chunk) {
          const uint32_t buf = chunk & 1;
          const bool bad = !mbar_wait(acc_full + buf, (chunk >> 1) & 1) || *abort_flag != 0;
          if (ff_epi_bar_or(bad)) { stop = true; break; }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < NA; c += 16) {
            float v[16];
            const int col = c < HC ? half * HC + c : BN_OUT + half * HC + c - HC;
            tmem_ld16_async(tmem_base + lanes + buf * BN + col, v);
            tmem_wait16(v);
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[c + e] += v[e];
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CG == 2) mbar_arrive_cluster(map_rank(acc_empty + buf, 0));
            else mbar_arrive(acc_empty + buf);
          }
        }
        if (!stop && row < g.M) {
#pragma unroll
          for (int c = 0; c < HC; c += 16)
            if (n0 + c < g.N) {
              float zg[16], zu[16];
              if (KIND == FF_DGATE) ff_load_z(g, row, n0 + c, zg, zu);
              ff_epilogue16<S, KIND>(g, m_part, row, n0 + c, acc + c, acc + (KIND == FF_GATE ? HC + c : c), zg, zu);
            }
        }
      } else {
        const uint32_t buf = chunk & 1;
        constexpr int CH = KIND == FF_DGATE && HC >= 32 ? 32 : 16;     // dgate: 16 loads of 32 bytes in flight per thread
        const bool bad = !mbar_wait(acc_full + buf, (chunk >> 1) & 1) || *abort_flag != 0;
        if (ff_epi_bar_or(bad)) stop = true;
        else {
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HC; c += CH) {
            float v[CH], u[16], zg[CH], zu[CH];
            if (KIND == FF_DGATE && row < g.M) {
#pragma unroll
              for (int e = 0; e < CH; e += 16)
                if (n0 + c + e < g.N) ff_load_z(g, row, n0 + c + e, zg + e, zu + e);
            }
#pragma unroll
            for (int e = 0; e < CH; e += 16) tmem_ld16_async(tmem_base + lanes + buf * BN + half * HC + c + e, v + e);
            if (KIND == FF_GATE) tmem_ld16_async(tmem_base + lanes + buf * BN + BN_OUT + half * HC + c, u);
#pragma unroll
            for (int e = 0; e < CH; e += 16) tmem_wait16(v + e);
            if (KIND == FF_GATE) tmem_wait16(u);
            if (row < g.M) {
#pragma unroll
              for (int e = 0; e < CH; e += 16)
                if (n0 + c + e < g.N) ff_epilogue16<S, KIND>(g, m_part, row, n0 + c + e, v + e, u, zg + e, zu + e);
            }
          }
          // the accumulator may be overwritten by the tile after next
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CG == 2) mbar_arrive_cluster(map_rank(acc_empty + buf, 0));
            else mbar_arrive(acc_empty + buf);
          }
          ++chunk;
        }
      }
      if (stop) { *abort_flag = 1; break; }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_all();    // the peer neither reads this CTA's shared memory nor signals its barriers any more
  if (threadIdx.x == 0 && *abort_flag) atomicExch(&g_ffn_error, 1);
  if (warp == 0) {
    tc_fence_after();
    ff_tmem_free<CG>(tmem_base, TMEM_COLS);
  }
}

// ---- operands: fp32 into three bf16 planes, 16-bit rows onto 32-byte boundaries -------------------------------------
// src [rows, cols] with lds elements per row -> dst [S][rows][ldd], ldd a multiple of sixteen; the tail columns are zero
// (uint16_t stands for either 16-bit type: the values are moved, not read)
__device__ __forceinline__ float to_f(uint16_t) { return 0.f; }
template <typename T, int S>
__global__ void __launch_bounds__(256) ffn_operand_kernel(const T* src, long long rows, int cols, long long lds, uint16_t* dst, int ldd) {
  pdl_wait();
  pdl_trigger();
  const int per_row = ldd / 8;
  const long long total = rows * per_row;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long r = i / per_row;
    const int c = (int)(i - r * per_row) * 8;
    const T* p = src + r * lds + c;
    uint16_t* q = dst + r * ldd + c;
    if (S == 3) {
      uint32_t o[3][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float lo[3], hi[3];
        split3(c + 2 * e < cols ? to_f(p[2 * e]) : 0.f, lo);
        split3(c + 2 * e + 1 < cols ? to_f(p[2 * e + 1]) : 0.f, hi);
#pragma unroll
        for (int s = 0; s < 3; ++s) o[s][e] = pack2(lo[s], hi[s], 0);
      }
#pragma unroll
      for (int s = 0; s < 3; ++s) *reinterpret_cast<uint4*>(q + s * rows * ldd) = make_uint4(o[s][0], o[s][1], o[s][2], o[s][3]);
    } else {
      Vec<T, 16 / sizeof(T)> v;
      v.clear();
#pragma unroll
      for (int e = 0; e < 16 / (int)sizeof(T); ++e)
        if (c + e < cols) v.e[e] = p[e];
      v.store(reinterpret_cast<T*>(q));
    }
  }
}

// ---------------------------------- host side ----------------------------------------------
static inline int pad16(int n) { return (n + 15) / 16 * 16; }

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

template <int BN, int S, int KIND, int CG>
static int ffn_launch_t(FfnGemm& g, const FfnOperand& a, const FfnOperand& b, cudaStream_t st) {
  void (*kernel)(FfnGemm) = ffn_gemm_kernel<BN, S, KIND, CG>;
  constexpr int smem = FfnSmem<BN, S, CG>::BYTES;
  // before the tensor maps: a runtime call makes the device's context current in a thread that has not used it yet
  // (autograd's), without which the driver refuses to encode a map
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return (int)e;
  int rc = ffn_map(&g.a, a, g.fp16, g.a_mn, FF_BM);
  if (rc) return rc;
  rc = ffn_map(&g.b, b, g.fp16, g.b_mn, KIND == FF_GATE ? BN / 2 : BN / CG);
  if (rc) return rc;
  const int bn_out = KIND == FF_GATE ? BN / 2 : BN;
  const long long tiles = (long long)((g.M + CG * FF_BM - 1) / (CG * FF_BM)) * g.m_parts * ((g.N + bn_out - 1) / bn_out);
  if (tiles > 0x3fffffffLL) return -1;
  const int most = sm_count() / CG, grid = CG * (tiles < most ? (int)tiles : most);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(FF_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (CG == 2) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = CG;
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
  return (int)cudaLaunchKernelEx(&cfg, kernel, g);
}

// Tile by the number of tiles: the widest that still gives every SM (pair) one (a narrow tile reads more operand bytes per
// multiplication; an idle SM costs more).
template <int S, int KIND>
static int ffn_launch(FfnGemm& g, const FfnOperand& a, const FfnOperand& b, cudaStream_t st) {
  const int cols = KIND == FF_GATE ? 2 * g.N : g.N, pairs = sm_count() / 2;
  const long long m2 = (long long)((g.M + 2 * FF_BM - 1) / (2 * FF_BM)) * g.m_parts;
  if (m2 * ((cols + 255) / 256) >= pairs) return ffn_launch_t<256, S, KIND, 2>(g, a, b, st);
  if (m2 * ((cols + 127) / 128) >= pairs) return ffn_launch_t<128, S, KIND, 2>(g, a, b, st);
  const long long m = (long long)((g.M + FF_BM - 1) / FF_BM) * g.m_parts;
  if (m * ((cols + 127) / 128) >= sm_count()) return ffn_launch_t<128, S, KIND, 1>(g, a, b, st);
  return ffn_launch_t<64, S, KIND, 1>(g, a, b, st);
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
  o->ld = pad16(cols);
  if (src == nullptr) return 0;       // prepared by the forward pass
  const long long runs = rows * (pad16(cols) / 8);
  const long long blocks = (runs + 255) / 256, most = 16LL * sm_count();
  const dim3 grid((unsigned)(blocks < most ? blocks : most)), block(256);
  const int ldd = pad16(cols);
  if (dt == DT_F32)
    return (int)launch_k(ffn_operand_kernel<float, 3>, grid, block, 0, st, (const float*)src, rows, cols, ld, (uint16_t*)dst, ldd);
  return (int)launch_k(ffn_operand_kernel<uint16_t, 1>, grid, block, 0, st, (const uint16_t*)src, rows, cols, ld, (uint16_t*)dst, ldd);
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
  const uintptr_t bits = (uintptr_t)out | (uintptr_t)(ldo * dt_bytes(dt));
  g.vec_bytes = bits % 32 == 0 ? 32 : (bits % 16 == 0 ? 16 : 0);
}

// Every operand comes with an optional image: [S][rows][pad16(cols)] 16-bit elements, S = 3 for fp32, needed for fp32 and
// for rows that do not start on 16-byte boundaries.  h: [S][m][pad16(f)] 16-bit; z: [2][m][pad16(f)] fp32 or null.
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
  g.out = h; g.ldo = pad16(f); g.z = z; g.ldz = pad16(f);
  rc = ffn_gemm<FF_GATE>(S, g, ox, oi, st);
  if (rc) return rc;
  const FfnOperand oh = {h, m, f, 1, S, pad16(f)};
  g.b_parts = 1;
  g.N = n; g.k_blocks = (f + FF_BK - 1) / FF_BK;
  ffn_out(g, y, dt, n);
  return ffn_gemm<FF_PLAIN>(S, g, oh, oo, st);
}

// x, w_in, w_out: as in the forward pass; where an image is given it holds the forward pass' image already.
// dz: [S][2][m][pad16(f)] 16-bit scratch.  dx, dw_in, dw_out may be null.
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
  const FfnOperand oh = {h, m, f, 1, S, pad16(f)}, oz = {dz, m, f, 2, S, pad16(f)};
  FfnGemm base = {};
  base.fp16 = dt == DT_F16;
  base.act = act;
  base.segments = base.m_parts = base.a_parts = base.b_parts = 1;
  FfnGemm g = base;
  if (dx != nullptr || dw_in != nullptr) {
    g.M = m; g.N = f; g.k_blocks = (n + FF_BK - 1) / FF_BK; g.b_mn = 1;
    g.out = dz; g.ldo = pad16(f); g.z = const_cast<float*>(z); g.ldz = pad16(f);
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
