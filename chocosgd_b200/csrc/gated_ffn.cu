// Gated feed-forward block on the 5th-generation tensor cores, forward and backward.
//
//   [G | U] = X W_in^T     W_in [2 F, D], gate rows first        H = act(G) * U            Y = H W_out^T      W_out [N, F]
//   dH = dY W_out          dG = dH U act'(G),  dU = dH act(G)    dX = dG W_in[:F] + dU W_in[F:]
//   dW_in = [dG | dU]^T X                                        dW_out = dY^T H
//
// Six products of one kernel (ffn_gemm_kernel), in four launches (the last three are independent of each other and share one, so
// that the tiles of all three fill the machine together), which differ in the operands' orientation and in the epilogue:
//   gate    both projections of a tile in ONE accumulator (the B tile holds BN / 2 gate rows and the BN / 2 up rows
//           that belong to them); the epilogue applies activation and product, so G and U meet in registers
//   dgate   dH stays in the accumulator: the epilogue reads G and U and writes dG and dU
//   plain   the four others
// No operand is ever transposed in memory: a tile is fetched K-major or MN-major, whichever way the tensor lies.
//
// Pipeline: one TMA thread, one thread that issues tcgen05.mma (kind::f16, fp32 accumulators in TMEM), eight or
// sixteen epilogue warps; operands in a ring of 128-byte-swizzled stages of 64 k, accumulators double-buffered so that the epilogue of a tile
// runs under the multiplications of the next (persistent CTAs).  Large products run as pairs of CTAs (cta_group::2, 256-row
// tiles): each CTA fetches half of the B tile, which halves its share of the operand traffic.
//
// Precision.  bf16 / fp16: operands as they are, fp32 accumulators; H and [dG | dU] are rounded once to the operands' type,
// because the next product reads them as tensor-core operands; G and U are kept in fp32 for the backward pass.
// fp32: every operand is the sum of three bf16 numbers (x = x1 + x2 + x3, each the rounded remainder of the ones before:
// 24 significant bits), a product is a1 b1 + (a1 b2 + a2 b1) + (a1 b3 + a2 b2 + a3 b1), what is left out is below 2^-24 of
// it.  The tensor core truncates when it adds to its accumulator, which over a long K costs far more than that
// (measured, one pass of exactly representable operands: relative error 7e-8 at K = 64, 4.4e-6 at K = 2600), so the fp32
// form takes its accumulator out after every 32 k and adds it up in registers; within those the small products go first.
// The whole operator at 1120 x 650 x 2600: 2.5e-7 off 64 bits, the same in fp32 arithmetic 9e-7 to 1.5e-6 (with 64 k per
// accumulator 8.5e-7, and 5 % less time).
//
// Bound by the tensor cores: 8192 x 2048 x 8192 bf16, gate 403 us (1.36 PFLOP/s), Y 191 (1.44), dgate 253 (1.09: it reads 0.5 GB
// of G and U and writes 0.27 GB), the three gradient products 924 (1.49); the library's plain products of the same sizes take 352,
// 178, 175 and 882 us without activation, G, U or their gradients.  fp32, 1120 x 650 x 2600: gate 52 us, Y 33 + 6, dgate 48, the
// gradients 125 + 8, images 16; there the epilogue, which takes the accumulator out every 32 k, costs as much as the products.
//
// Every mbarrier wait is bounded.  A wait that runs out ends the work of its CTA (both CTAs of a pair): results that are not written by
// then stay unwritten, the copies and multiplications in flight are waited for, TMEM is freed and the error word is set.
#include "block_calls.h"
#include "launch.cuh"
#include "tc_common.cuh"
#include "ffn.cuh"

#include <atomic>

#define FF_BM 128            // accumulator rows of one CTA
#define FF_BK(S) ((S) == 3 ? 32 : 64)    // k per stage: K-major rows of 64 (three planes) or 128 bytes = one swizzle row
// epilogue warps 0 .. EPI - 1 (warp 0 owns TMEM), then the TMA warp and the MMA warp
#define FF_THREADS(EPI) (32 * ((EPI) + 2))

#define FF_GATE 0
#define FF_DGATE 1
#define FF_PLAIN 2           // also over a part of k, into fp32 slices that ffn_join_kernel adds up (k_splits > 1)

__device__ int g_ffn_error;

struct FfnGemm {
  CUtensorMap a, b;
  int M, N;              // output rows (of one part) and columns; gate: N = F
  int k_blocks;          // k-blocks (FF_BK) of one segment
  int k_splits;          // plain: slices of the k-blocks, one tile each (1: the result itself)
  int segments;          // dX: 2 (gate and up rows of W_in); else 1
  int m_parts;           // dW_in: 2 (dG and dU); else 1
  int a_parts, b_parts;  // planes per split of the operand (2: gate / up)
  int a_mn, b_mn;        // operand lies MN-major
  int fp16;              // operand type: fp16 instead of bf16 (S = 1)
  int act;
  void* out;             // plain: [m_parts M, N] of the operands' type;  gate: H [S][M][ldo];  dgate: dZ [S][2][M][ldo]
  int vec16;             // out's rows start on 16-byte boundaries
  long long ldo;
  float* z;              // lane-blocked fp32 (lane_off), ldz columns.  gate: [2] G, U written (null in evaluation);
  long long ldz;         // dgate: read;  plain in slices: [k_splits][m_parts] written
  long long z_plane;     // floats of one matrix of z
};

// products of one launch: tiles first[i] .. first[i + 1] - 1 are those of g[i] (gate, dgate: one product)
struct FfnBatch {
  FfnGemm g[3];
  int n, first[4];
  int give_up;           // not 0 (tests): CTAs of the ranks in bits 0 and 1 act after (give_up >> 2) ns as if a wait had run out
};

// fp32 matrices that only these kernels read (G, U, partial sums) are stored in the order in which a warp of the epilogue
// holds them: 32 rows x 8 columns = 1 KB, 32 bytes per lane.  Row-major, a warp's access would touch 32 lines for 1 KB.
__host__ __device__ __forceinline__ long long lane_off(int row, int col, long long ld) {
  return (((long long)(row >> 5) * (ld >> 3) + (col >> 3)) * 32 + (row & 31)) * 8;
}

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
// as mbar_wait, and false too once the CTA (or its peer) has given up
__device__ __forceinline__ bool ff_wait(uint64_t* bar, uint32_t parity, const volatile int* abort_flag) {
  const uint32_t addr = smem_u32(bar);
  for (uint32_t i = 0; i < SPIN_LIMIT; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(addr), "r"(parity) : "memory");
    if (ok) return true;
    if (i > 1024) {
      if (*abort_flag != 0) return false;
      __nanosleep(64);
    }
  }
  return false;
}
// ends the work of this CTA, and of its peer
template <int CG>
__device__ __forceinline__ void ff_give_up(volatile int* abort_flag, uint32_t rank) {
  *abort_flag = 1;
  if (CG == 2)
    asm volatile("st.volatile.shared::cluster.u32 [%0], %1;" ::"r"(map_rank(const_cast<const int*>(abort_flag), rank ^ 1)), "r"(1) : "memory");
}
template <int EPI>
__device__ __forceinline__ bool ff_epi_bar_or(bool flag) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, 1, %2, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r) : "r"((uint32_t)flag), "n"(EPI * 32) : "memory");
  return r != 0;
}

// a word of the peer's shared memory
__device__ __forceinline__ uint32_t ff_peer_word(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.volatile.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void ff_complete_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
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

// ---- a warp's 32 rows x up to 128 bytes through shared memory, so that rows are written as whole lines -----------------
// 16-byte unit c of row r lies at unit c ^ (r & 7) of the row's 128 bytes
__device__ __forceinline__ void stage_put(uint8_t* stage, int lane, int unit, uint4 v) {
  *reinterpret_cast<uint4*>(stage + lane * 128 + ((unit ^ (lane & 7)) << 4)) = v;
}
__device__ __forceinline__ uint4 stage_get(const uint8_t* stage, int row, int unit) {
  return *reinterpret_cast<const uint4*>(stage + row * 128 + ((unit ^ (row & 7)) << 4));
}
// UNITS 16-byte units per row, from unit `u0`, to rows [0, rows) of `out` (ES bytes per element, ld elements per row), of
// which `cols` elements exist.  vec16: rows start on 16-byte boundaries.  Called by whole warps.
template <int UNITS, int ES>
__device__ __forceinline__ void stage_flush(const uint8_t* stage, int u0, uint8_t* out, long long ld, int rows, int cols,
                                            int vec16, int lane) {
  constexpr int EU = 16 / ES;      // elements per unit
  if (vec16) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const int r = (i * 32 + lane) / UNITS, c = (i * 32 + lane) % UNITS;
      if (r < rows && c * EU < cols) {
        const uint4 v = stage_get(stage, r, u0 + c);
        uint8_t* p = out + ((long long)r * ld + c * EU) * ES;
        if (c * EU + EU <= cols) {
          *reinterpret_cast<uint4*>(p) = v;
        } else {
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < EU; ++e)
            if (c * EU + e < cols) {
              if (ES == 4) reinterpret_cast<uint32_t*>(p)[e] = w[e & 3];
              else reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
            }
        }
      }
    }
  } else {
#pragma unroll 1
    for (int r = 0; r < rows; ++r) {
#pragma unroll
      for (int e = lane; e < UNITS * EU; e += 32)
        if (e < cols) {
          const uint8_t* src = stage + r * 128 + (((u0 + e / EU) ^ (r & 7)) << 4) + (e % EU) * ES;
          uint8_t* p = out + ((long long)r * ld + e) * ES;
          if (ES == 4) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(src);
          else *reinterpret_cast<uint16_t*>(p) = *reinterpret_cast<const uint16_t*>(src);
        }
    }
  }
}

// What a warp does with its 32 rows x HC output columns of a tile, sixteen columns at a time: put() for each, in order.
// v = accumulator (gate: G in v, U in u; dgate: dH, with G and U in zg, zu).  Buffers between the products have rows padded
// to sixteen elements and are written in whole runs.
template <int S, int KIND, int HC, int ACT> struct FfnEpilogue {
  const FfnGemm& g;
  uint8_t* stage;
  int m_part, row0, col0, lane;      // first row and column of the warp
  float* z;                          // this lane's place of (row0, col0) in z; 16 columns are 512 floats

  __device__ __forceinline__ void put(int c, const float* v, const float* u, const float* zg, const float* zu) {
    constexpr bool FAST = S == 1;
    const int col = col0 + c;
    if (KIND == FF_GATE) {
      float h[16], slope;
      if (g.z != nullptr && row0 < g.M && col < g.N) {
        float *zg_at = z + c * 32, *zu_at = zg_at + g.z_plane;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          st32b(zg_at + k * 256, reinterpret_cast<const uint32_t*>(v + 8 * k));
          st32b(zu_at + k * 256, reinterpret_cast<const uint32_t*>(u + 8 * k));
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) h[e] = ff_act<ACT, false, FAST>(v[e], slope) * u[e];
      operand<(HC < 64 ? HC : 64)>(c, 0, h, 0, g.M * g.ldo);
    } else if (KIND == FF_DGATE) {
      float dg[16], du[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float slope;
        const float a = ff_act<ACT, true, FAST>(zg[e], slope);
        du[e] = v[e] * a;
        dg[e] = v[e] * zu[e] * slope;
      }
      const long long plane = g.M * g.ldo;
      operand<(HC < 32 ? HC : 32)>(c, 0, dg, 0, 2 * plane);
      operand<(HC < 32 ? HC : 32)>(c, 4, du, plane, 2 * plane);
    } else if (g.k_splits > 1) {
      if (row0 < g.M && col < g.N) {
        st32b(z + c * 32, reinterpret_cast<const uint32_t*>(v));
        st32b(z + c * 32 + 256, reinterpret_cast<const uint32_t*>(v + 8));
      }
    } else if (S == 3) {
      constexpr int FC = HC < 32 ? HC : 32;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        stage_put(stage, lane, c % FC / 4 + k, make_uint4(__float_as_uint(v[4 * k]), __float_as_uint(v[4 * k + 1]),
                                                          __float_as_uint(v[4 * k + 2]), __float_as_uint(v[4 * k + 3])));
      if ((c + 16) % FC == 0) flush<FC / 4, 4>(c + 16 - FC, 0, (long long)m_part * g.M * g.ldo, g.N);
    } else {
      constexpr int FC = HC < 64 ? HC : 64;
      pack16(c % FC / 8, v);
      if ((c + 16) % FC == 0) flush<FC / 8, 2>(c + 16 - FC, 0, (long long)m_part * g.M * g.ldo, g.N);
    }
  }
  __device__ __forceinline__ void pack16(int unit, const float* v) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      stage_put(stage, lane, unit + k, make_uint4(pack2(v[8 * k], v[8 * k + 1], g.fp16), pack2(v[8 * k + 2], v[8 * k + 3], g.fp16),
                                                  pack2(v[8 * k + 4], v[8 * k + 5], g.fp16), pack2(v[8 * k + 6], v[8 * k + 7], g.fp16)));
  }
  template <int UNITS, int ES>
  __device__ __forceinline__ void flush(int c, int u0, long long off, long long cols) {
    __syncwarp();
    stage_flush<UNITS, ES>(stage, u0, reinterpret_cast<uint8_t*>(g.out) + (off + (long long)row0 * g.ldo + col0 + c) * ES, g.ldo,
                           min(32, g.M - row0), (int)cols - col0 - c, g.vec16, lane);
    __syncwarp();
  }
  // a 16-bit operand buffer: FC columns are gathered in shared memory (from unit u0); three planes are written directly
  template <int FC>
  __device__ __forceinline__ void operand(int c, int u0, const float* v, long long off, long long plane) {
    if (S == 3) {
      if (row0 + lane >= g.M || col0 + c >= g.ldo) return;
      uint32_t q[3][8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t p[3];
        split3(v[2 * e], v[2 * e + 1], p);
#pragma unroll
        for (int s = 0; s < 3; ++s) q[s][e] = p[s];
      }
      uint16_t* o = reinterpret_cast<uint16_t*>(g.out) + off + (long long)(row0 + lane) * g.ldo + col0 + c;
#pragma unroll
      for (int s = 0; s < 3; ++s) st32b(o + s * plane, q[s]);
    } else {
      pack16(u0 + c % FC / 8, v);
      if ((c + 16) % FC == 0) flush<FC / 8, 2>(c + 16 - FC, u0, off, g.ldo);
    }
  }
};
// G and U of sixteen columns of a row (dgate) from this lane's place in z; zeros outside
__device__ __forceinline__ void ff_load_z(const float* z, long long z_plane, bool inside, float* zg, float* zu) {
  if (inside) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      ld32b(z + k * 256, reinterpret_cast<uint32_t*>(zg + 8 * k));
      ld32b(z + z_plane + k * 256, reinterpret_cast<uint32_t*>(zu + 8 * k));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) zg[e] = zu[e] = 0.f;
  }
}

// BN accumulator columns, S operand planes, CG CTAs per tile: a pair (CG = 2) shares one 256-row tile, each CTA fetches its
// 128 rows of A and half of the B tile, so a byte of B serves 256 rows
template <int BN, int S, int KIND, int CG> struct FfnSmem {
  // Epilogue warps.  Three planes: the sums of a tile end in the epilogue's registers, so it does not run under the next tile;
  // with sixteen warps its activation and splitting take less (1120 x 650 x 2600, gate 51.8 -> 47.8 us, dgate 52.4 -> 44.8).
  // 16-bit operands: eight (dgate at 8192 x 2048 x 8192: 259 us, with sixteen and no room to fetch ahead 273).
  static constexpr int EPI = S == 3 && (KIND == FF_DGATE || (KIND == FF_GATE && BN >= 128) || BN == 256) ? 16 : 8;
  static constexpr int A_TILE = FF_BM * FF_BK(S) * 2, B_TILE = BN / CG * FF_BK(S) * 2;
  static constexpr int STAGE = S * (A_TILE + B_TILE);
  static constexpr int EPI_BYTES = EPI * 4096;            // 4 KB for each epilogue warp
  static constexpr int ROOM = 227 * 1024 - 256 - 1024 - EPI_BYTES;
  static constexpr int STAGES = ROOM / STAGE > 8 ? 8 : ROOM / STAGE;
  static_assert((2 * STAGES + 5) * 8 + 12 <= 256, "barriers and words");
  static constexpr int BYTES = STAGES * STAGE + EPI_BYTES + 256 + 1024;
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

// f(the activation as a constant): the choice is made once per tile, so that the code that runs stays small
template <int V> struct FfnConst { static constexpr int value = V; };
template <int KIND, typename F>
__device__ __forceinline__ void ff_for_act(int act, F f) {
  if (KIND == FF_PLAIN || act == ACT_SILU) f(FfnConst<ACT_SILU>());
  else if (act == ACT_GELU) f(FfnConst<ACT_GELU>());
  else if (act == ACT_RELU) f(FfnConst<ACT_RELU>());
  else f(FfnConst<ACT_SIGMOID>());
}

// where a tile lies: its product, its first output row and column, its part and slice, its k-blocks [kb0, kb1)
template <int BN_OUT, int TM, int KIND> struct FfnWhere {
  const FfnGemm& g;
  int m0, n0, m_part, slice, kb0, kb1;
  static __device__ __forceinline__ int which(const FfnBatch& b, int tile) {
    int i = 0;
    if (KIND == FF_PLAIN)
      while (i + 1 < b.n && tile >= b.first[i + 1]) ++i;
    return i;
  }
  __device__ __forceinline__ FfnWhere(const FfnBatch& b, int tile, int i) : g(b.g[i]) {
    const int tiles_m = (g.M + TM - 1) / TM, tiles_n = (g.N + BN_OUT - 1) / BN_OUT, out_tiles = tiles_m * g.m_parts * tiles_n;
    int local = tile - b.first[i], tm, tn;
    slice = KIND == FF_PLAIN ? local / out_tiles : 0;
    local -= slice * out_tiles;
    ff_tile(local, tiles_m * g.m_parts, tiles_n, tm, tn);
    m_part = tm / tiles_m;
    m0 = (tm - m_part * tiles_m) * TM;
    n0 = tn * BN_OUT;
    const int n_kb = g.k_blocks * g.segments;
    kb0 = KIND == FF_PLAIN ? (int)((long long)n_kb * slice / g.k_splits) : 0;
    kb1 = KIND == FF_PLAIN ? (int)((long long)n_kb * (slice + 1) / g.k_splits) : n_kb;
  }
};

template <int BN, int S, int KIND, int CG>
__global__ void __launch_bounds__(FF_THREADS((FfnSmem<BN, S, KIND, CG>::EPI)), 1) ffn_gemm_kernel(const __grid_constant__ FfnBatch batch) {
  typedef FfnSmem<BN, S, KIND, CG> L;
  extern __shared__ uint8_t smem_raw[];
  // 1024-byte alignment: the swizzle pattern is a function of the shared-memory address bits
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int BK = FF_BK(S);
  uint8_t* epi_smem = smem + L::STAGES * L::STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(epi_smem + L::EPI_BYTES);   // CG = 2: the leader's count both CTAs' bytes
  uint64_t* empty = full + L::STAGES;
  uint64_t* acc_full = empty + L::STAGES;    // [2]
  uint64_t* acc_empty = acc_full + 2;        // [2], the leader's
  uint64_t* drained = acc_empty + 2;         // after a wait that ran out
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* issued = tmem_slot + 2; // stages that this CTA's copies were started for
  constexpr int BN_OUT = KIND == FF_GATE ? BN / 2 : BN;    // output columns of a tile
  constexpr int TM = FF_BM * CG;                           // output rows of a tile

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  typedef FfnWhere<BN_OUT, TM, KIND> Where;
  const int n_tiles = batch.first[batch.n];
  const int first_tile = blockIdx.x / CG, tile_step = gridDim.x / CG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full + b, 1);
      mbar_init(acc_empty + b, L::EPI * CG);   // one arrival per epilogue warp
    }
    mbar_init(drained, 1);
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
  if (warp == L::EPI) {
    // ---------------- TMA producer ----------------
    uint32_t it = 0, s = 0, phase = 1;      // stage and the parity of its `empty` barrier (the first round passes at once)
    bool ok = true;
    for (int tile = first_tile; tile < n_tiles && ok; tile += tile_step) {
      const Where at(batch, tile, Where::which(batch, tile));
      const FfnGemm& g = at.g;
      const int n0 = at.n0, m_part = at.m_part, m0 = at.m0 + (int)rank * FF_BM;
      {
        for (int i = at.kb0; i < at.kb1; ++i) {
          const int seg = i >= g.k_blocks ? 1 : 0, k0 = (i - seg * g.k_blocks) * BK;
          const int part_a = g.m_parts > 1 ? m_part : (g.a_parts > 1 ? seg : 0), part_b = g.b_parts > 1 ? seg : 0;
          ok = __all_sync(0xffffffffu, ff_wait(empty + s, phase, abort_flag) && *abort_flag == 0);
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
                for (int j = 0; j < FF_BM / 64; ++j) tma_load_3d<CG>(dA + j * BK * 128, &g.a, bar, m0 + 64 * j, k0, pa);
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
                  for (int j = 0; j < BN / CG / 64; ++j) tma_load_3d<CG>(dB + j * BK * 128, &g.b, bar, nb + 64 * j, k0, pb);
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
    if (lane == 0) *issued = it;
    if (!ok) ff_give_up<CG>(abort_flag, rank);
  } else if (warp == L::EPI + 1 && rank == 0) {
    // ---------------- MMA issuer (of a pair: the leader's) ----------------
    uint32_t s = 0, phase = 0, chunk = 0;
    const uint32_t base = smem_u32(smem);
    bool ok = true;
    for (int tile = first_tile; tile < n_tiles && ok; tile += tile_step) {
      const Where at(batch, tile, Where::which(batch, tile));
      const FfnGemm& g = at.g;
      const int n_kb = at.kb1 - at.kb0;
      // instruction descriptor: fp32 accumulate, operand type, majorness bits, N >> 3, M >> 4
      const uint32_t type = g.fp16 ? 0u : 1u;
      const uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)g.a_mn << 15) | ((uint32_t)g.b_mn << 16) |
                             ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
      // K-major: 16 k = 32 bytes further inside the (64- or 128-byte) row, groups of 8 rows apart; MN-major: 16 k = 16 rows of
      // 128 bytes, 8-k groups 1024 bytes apart, blocks of 64 MN elements BK rows apart.  Descriptors count in 16 bytes.
      const uint32_t a_step = (g.a_mn ? 2048 : 32) >> 4, b_step = (g.b_mn ? 2048 : 32) >> 4;
      const uint64_t da0 = g.a_mn ? make_desc(base, BK * 128, 1024) : make_desc(base, 16, BK * 16, BK == 32 ? 4 : 2);
      const uint64_t db0 = g.b_mn ? make_desc(base + S * L::A_TILE, BK * 128, 1024)
                                  : make_desc(base + S * L::A_TILE, 16, BK * 16, BK == 32 ? 4 : 2);
      for (int i = 0; i < n_kb; ++i) {
        const uint32_t buf = chunk & 1;
        const bool first = S == 3 || i == 0, last = S == 3 || i == n_kb - 1;      // S = 3: every k-block has its accumulator
        // the first round of either accumulator passes at once
        if (first) ok = ff_wait(acc_empty + buf, ((chunk >> 1) & 1) ^ 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok && ff_wait(full + s, phase, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t d = tmem_base + buf * BN;
          const uint64_t da = da0 + s * (L::STAGE >> 4), db = db0 + s * (L::STAGE >> 4);
          if (S == 1) {
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) umma_f16<CG>(d, da + k * a_step, db + k * b_step, idesc, (!first || k > 0) ? 1u : 0u);
          } else {
            // smallest products first: (1,3) (3,1) (2,2) (1,2) (2,1) (1,1)
            constexpr int PA[6] = {0, 2, 1, 0, 1, 0}, PB[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
            for (int p = 0; p < 6; ++p)
#pragma unroll
              for (int k = 0; k < BK / 16; ++k)
                umma_f16<CG>(d, da + PA[p] * (L::A_TILE >> 4) + k * a_step, db + PB[p] * (L::B_TILE >> 4) + k * b_step, idesc,
                             (!first || p > 0 || k > 0) ? 1u : 0u);
          }
          ff_commit<CG>(empty + s);  // frees this stage once the MMAs above have read it
          if (last) ff_commit<CG>(acc_full + buf);
        }
        __syncwarp();
        if (last) ++chunk;
        if (++s == L::STAGES) { s = 0; phase ^= 1; }
      }
    }
    if (!ok) ff_give_up<CG>(abort_flag, rank);
  } else if (warp < L::EPI) {
    // ---------------- epilogue: warp w reads lanes 32 (w % 4) ... of its share of the tile's output columns ----------------
    constexpr int HC = BN_OUT / (L::EPI / 4);         // output columns per warp
    const int half = warp >> 2;
    uint32_t chunk = 0;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    if (batch.give_up != 0 && threadIdx.x == 0 && (batch.give_up >> rank & 1)) {
      __nanosleep((uint32_t)batch.give_up >> 2);
      ff_give_up<CG>(abort_flag, rank);
    }
    for (int tile = first_tile; tile < n_tiles; tile += tile_step) {
      const Where at(batch, tile, Where::which(batch, tile));
      const FfnGemm& g = at.g;
      const int m_part = at.m_part;
      const int row0 = at.m0 + (int)rank * FF_BM + (warp & 3) * 32, col0 = at.n0 + half * HC;
      float* z = nullptr;
      if (g.z != nullptr)
        z = g.z + (KIND == FF_PLAIN ? (at.slice * g.m_parts + m_part) * g.z_plane : 0) + lane_off(row0 + lane, col0, g.ldz);
      const int z_cols = row0 < g.M ? g.N - col0 : 0;      // columns of z that exist
      bool stop = false;
      if (S == 3) {
        // the accumulators of all k-blocks, added up in registers
        constexpr int NA = KIND == FF_GATE ? 2 * HC : HC;
        float acc[NA];
#pragma unroll
        for (int c = 0; c < NA; ++c) acc[c] = 0.f;
        for (int i = at.kb0; i < at.kb1; ++i, ++chunk) {
          const uint32_t buf = chunk & 1;
          const bool bad = !ff_wait(acc_full + buf, (chunk >> 1) & 1, abort_flag) || *abort_flag != 0;
          if (ff_epi_bar_or<L::EPI>(bad)) { stop = true; break; }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < NA; c += 32) {
            float v[32];
#pragma unroll
            for (int e = 0; e < 32 && c + e < NA; e += 16) {
              const int col = c + e < HC ? half * HC + c + e : BN_OUT + half * HC + c + e - HC;
              tmem_ld16_async(tmem_base + lanes + buf * BN + col, v + e);
            }
#pragma unroll
            for (int e = 0; e < 32 && c + e < NA; e += 16) tmem_wait16(v + e);
#pragma unroll
            for (int e = 0; e < 32 && c + e < NA; ++e) acc[c + e] += v[e];
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CG == 2) mbar_arrive_cluster(map_rank(acc_empty + buf, 0));
            else mbar_arrive(acc_empty + buf);
          }
        }
        if (!stop) {
          ff_for_act<KIND>(g.act, [&](auto act) {
            FfnEpilogue<S, KIND, HC, decltype(act)::value> epi = {g, epi_smem + warp * 4096, m_part, row0, col0, lane, z};
            float zg[16], zu[16];
#pragma unroll
            for (int c = 0; c < HC; c += 16) {
              if (KIND == FF_DGATE) ff_load_z(z + c * 32, g.z_plane, c < z_cols, zg, zu);
              epi.put(c, acc + c, acc + (KIND == FF_GATE ? HC + c : c), zg, zu);
            }
          });
        }
      } else {
        const uint32_t buf = chunk & 1;
        // dgate: G and U of the next sixteen columns are under way while the present ones are worked on; the first ones
        // while the tile is still being multiplied
        float zg[16], zu[16], yg[16], yu[16];
        if (KIND == FF_DGATE) ff_load_z(z, g.z_plane, 0 < z_cols, zg, zu);
        const bool bad = !ff_wait(acc_full + buf, (chunk >> 1) & 1, abort_flag) || *abort_flag != 0;
        if (ff_epi_bar_or<L::EPI>(bad)) stop = true;
        else {
          tc_fence_after();
          ff_for_act<KIND>(g.act, [&](auto act) {
            FfnEpilogue<S, KIND, HC, decltype(act)::value> epi = {g, epi_smem + warp * 4096, m_part, row0, col0, lane, z};
            const uint32_t acc = tmem_base + lanes + buf * BN + half * HC;
#pragma unroll 1
            for (int c = 0; c < HC; c += 32) {
              float v[16], u[16];
              if (KIND == FF_DGATE && c + 16 < HC) ff_load_z(z + c * 32 + 512, g.z_plane, c + 16 < z_cols, yg, yu);
              tmem_ld16_async(acc + c, v);
              if (KIND == FF_GATE) tmem_ld16_async(acc + BN_OUT + c, u);
              tmem_wait16(v);
              if (KIND == FF_GATE) tmem_wait16(u);
              epi.put(c, v, u, zg, zu);
              if (HC < 32) break;
              if (KIND == FF_DGATE && c + 32 < HC) ff_load_z(z + c * 32 + 1024, g.z_plane, c + 32 < z_cols, zg, zu);
              tmem_ld16_async(acc + c + 16, v);
              if (KIND == FF_GATE) tmem_ld16_async(acc + BN_OUT + c + 16, u);
              tmem_wait16(v);
              if (KIND == FF_GATE) tmem_wait16(u);
              epi.put(c + 16, v, u, yg, yu);
            }
          });
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
      if (stop) {
        ff_give_up<CG>(abort_flag, rank);
        break;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_all();    // the peer neither reads this CTA's shared memory nor signals its barriers any more
  if (*abort_flag) {      // the same in both CTAs of a pair
    if (threadIdx.x == 0) atomicExch(&g_ffn_error, 1);
    if (warp == L::EPI && rank == 0) {
      // Copies: those of the last STAGES stages that either CTA has started.  One half of a pair's stage may not have been started;
      // the leader then counts for it: its arrival where its own is missing, the bytes of the peer's half where that one is.
      const uint32_t mine = *issued, peer = CG == 2 ? ff_peer_word(map_rank(const_cast<const uint32_t*>(issued), 1)) : mine;
      const uint32_t end = mine > peer ? mine : peer;
      for (uint32_t j = end > L::STAGES ? end - L::STAGES : 0; j < end; ++j) {
        uint64_t* bar = full + j % L::STAGES;
        if (CG == 2 && lane == 0) {
          if (j >= mine) mbar_expect_tx(bar, L::STAGE);
          if (j >= peer) ff_complete_tx(bar, L::STAGE);
        }
        __syncwarp();
        mbar_wait(bar, (j / L::STAGES) & 1);
      }
    }
    if (warp == L::EPI + 1) {
      if (rank == 0 && elect_one()) ff_commit<CG>(drained);
      __syncwarp();
      mbar_wait(drained, 0);
    }
    __syncthreads();
    if (CG == 2) cluster_sync_all();
  }
  if (warp == 0) {
    tc_fence_after();
    ff_tmem_free<CG>(tmem_base, TMEM_COLS);
  }
}

// ---- operands: fp32 into three bf16 planes, 16-bit rows onto 32-byte boundaries -------------------------------------
// src [rows, cols] with lds elements per row -> dst [S][rows][ldd], ldd a multiple of sixteen; the tail columns are zero
struct FfnImage {
  const void* src;
  uint16_t* dst;
  long long rows, lds;
  int cols, ldd, vec;       // vec: elements per access that the row starts allow (1, 2, 4)
  unsigned first_block;     // blocks [first_block, next image's) copy this matrix, eight elements per thread
};
struct FfnImages {
  FfnImage m[4];
  int n;
};
template <int S>
__global__ void __launch_bounds__(256) ffn_operand_kernel(const __grid_constant__ FfnImages a) {
  pdl_wait();
  pdl_trigger();
  int k = 0;
  while (k + 1 < a.n && blockIdx.x >= a.m[k + 1].first_block) ++k;
  const FfnImage& m = a.m[k];
  const unsigned per_row = m.ldd / 8, i = (blockIdx.x - m.first_block) * 256 + threadIdx.x;
  const long long r = i / per_row;
  const int c = (int)(i - (unsigned)r * per_row) * 8;
  if (r < m.rows) {
    uint16_t* q = m.dst + r * m.ldd + c;
    if (S == 3) {
      const float* p = reinterpret_cast<const float*>(m.src) + r * m.lds + c;
      float v[8];
      if (c + 8 <= m.cols && m.vec == 4) {
        *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p);
        *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(p + 4);
      } else if (c + 8 <= m.cols && m.vec == 2) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) *reinterpret_cast<float2*>(v + e) = *reinterpret_cast<const float2*>(p + e);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < m.cols ? p[e] : 0.f;
      }
      uint32_t o[3][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t w[3];
        split3(v[2 * e], v[2 * e + 1], w);
#pragma unroll
        for (int s = 0; s < 3; ++s) o[s][e] = w[s];
      }
#pragma unroll
      for (int s = 0; s < 3; ++s) *reinterpret_cast<uint4*>(q + s * m.rows * m.ldd) = make_uint4(o[s][0], o[s][1], o[s][2], o[s][3]);
    } else {
      // 16-bit values are moved, not read
      const uint16_t* p = reinterpret_cast<const uint16_t*>(m.src) + r * m.lds + c;
      Vec<uint16_t, 8> v;
      v.clear();
      if (c + 8 <= m.cols && m.vec >= 2) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = *reinterpret_cast<const uint32_t*>(p + 2 * e);
        v.raw = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < m.cols) v.e[e] = p[e];
      }
      v.store(q);
    }
  }
}

// out [m_parts M, N] = sum over k_splits slices of partial sums, in slice order.  A block takes 32 rows x 64 columns: eight
// warps read eight lane-blocked groups each slice, and rows are written as they lie in memory.
template <typename T>
__global__ void __launch_bounds__(256) ffn_join_kernel(const float* z, long long ldz, long long z_plane, int splits, int m_parts,
                                                       int M, int N, T* out) {
  __shared__ float tile[32][65];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, blocks = (M + 31) / 32;
  const int part = blockIdx.y / blocks, row0 = (blockIdx.y - part * blocks) * 32, col0 = blockIdx.x * 64;
  if (col0 + warp * 8 < ldz) {
    float v[8], w[8];
    const float* p = z + part * z_plane + lane_off(row0 + lane, col0 + warp * 8, ldz);
    ld32b(p, reinterpret_cast<uint32_t*>(v));
#pragma unroll 4
    for (int q = 1; q < splits; ++q) {
      ld32b(p + (long long)q * m_parts * z_plane, reinterpret_cast<uint32_t*>(w));
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += w[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) tile[lane][warp * 8 + e] = v[e];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int i = k * 256 + threadIdx.x, r = i >> 6, c = i & 63;
    if (row0 + r < M && col0 + c < N) out[((long long)part * M + row0 + r) * N + col0 + c] = from_f<T>(tile[r][c]);
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

static int ffn_map(CUtensorMap* map, const FfnOperand& o, int fp16, int mn_major, int box_rows, int bk) {
  TcEncodeTiledFn enc = tc_get_encode();
  if (enc == nullptr) return -10;
  if (((uintptr_t)o.p & 15) != 0 || o.ld % 8 != 0) return -11;
  cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)(o.parts * o.splits)};
  cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)o.ld * 2 * (cuuint64_t)o.rows};
  cuuint32_t box[3] = {(cuuint32_t)(mn_major ? 64 : bk), (cuuint32_t)(mn_major ? bk : box_rows), 1}, es[3] = {1, 1, 1};
  CUresult r = enc(map, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.p),
                   dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   !mn_major && bk == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -12;
}

struct FfnOperands {
  FfnOperand a, b;
};

// Launches of a call behind its first are programmatic dependents of the one before (all kernels wait before they touch global
// memory), unless they run for many tiles per SM (777 x 1111 x 2777 fp16, all launches of a training pass: 132 -> 127.6 us, 1120 x 650
// x 2600 fp32 274 -> 270; 8192 x 2048 x 8192 bf16 2170 -> 2206 with them, so not there).
struct FfnChain {
  int launches = 0;         // so far; every launch asks dependent() once
  bool dependent(bool few_tiles = true) {
    const bool d = (launches > 0 && few_tiles && pdl_in_call()) || pdl_enabled();
    ++launches;
    return d;
  }
};
static thread_local FfnChain ffn_chain;      // of the call that this thread is in

static std::atomic<int> ffn_give_up{0};
// for tests: `give_up` of the launches that follow (FfnBatch); returns the one before
extern "C" int gated_ffn_give_up(int how) { return ffn_give_up.exchange(how); }

template <int BN, int S, int KIND, int CG>
static int ffn_launch_t(FfnBatch& batch, const FfnOperands* o, cudaStream_t st) {
  void (*kernel)(FfnBatch) = ffn_gemm_kernel<BN, S, KIND, CG>;
  typedef FfnSmem<BN, S, KIND, CG> L;
  constexpr int smem = L::BYTES;
  // before the tensor maps: a runtime call makes the device's context current in a thread that has not used it yet
  // (autograd's), without which the driver refuses to encode a map
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return (int)e;
  const int bn_out = KIND == FF_GATE ? BN / 2 : BN;
  long long tiles = 0;
  for (int i = 0; i < batch.n; ++i) {
    FfnGemm& g = batch.g[i];
    int rc = ffn_map(&g.a, o[i].a, g.fp16, g.a_mn, FF_BM, FF_BK(S));
    if (rc) return rc;
    rc = ffn_map(&g.b, o[i].b, g.fp16, g.b_mn, KIND == FF_GATE ? BN / 2 : BN / CG, FF_BK(S));
    if (rc) return rc;
    batch.first[i] = (int)tiles;
    tiles += (long long)((g.M + CG * FF_BM - 1) / (CG * FF_BM)) * g.m_parts * ((g.N + bn_out - 1) / bn_out) * g.k_splits;
    if (tiles > 0x3fffffffLL) return -1;
  }
  batch.first[batch.n] = (int)tiles;
  batch.give_up = ffn_give_up;
  const int most = sm_count() / CG, grid = CG * (tiles < most ? (int)tiles : most);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(FF_THREADS(L::EPI));
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
  if (ffn_chain.dependent(tiles <= 4LL * most)) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return (int)cudaLaunchKernelEx(&cfg, kernel, batch);
}

// Which tile a launch runs with, by its time in SM cycles:  tiles per SM (pair) x (64-k blocks x step + exposed epilogue), where
//   step      16-bit operands: the slower of multiplying (1024 multiply-adds x 4 per cycle and SM) and of fetching the operands
//             (measured: about 58 bytes per cycle and SM from L2 when all SMs fetch); three planes: shared memory, from which every
//             one of the six products reads its operands (measured about 120 bytes per cycle: 2420 cycles at a width of 128, 3200 at 256)
//   epilogue  (measured) runs under the next tile's multiplications for 16-bit operands, not for three planes (whose sums are in
//             the epilogue's registers)
// One product: whole rounds.  Several: their tiles follow one another, so the average load and half of the largest tile.
// A plain product can be cut into slices of k, which costs the partial sums' second pass: a launch, then 4 bytes of each written and read.
struct FfnProduct {
  int M, m_parts, cols;
  long long k64;
};
struct FfnPlan {
  int bn, cg, splits[3];
};
static double ffn_tile_cost(int bn, int cg, int S, int kind, long long k64) {
  const double mul = 2.0 * bn, fetch = (FF_BM + bn / cg) * 128.0 / 58.0;
  // three planes: 24 multiplications of 16 k read (128 + bn) rows of 32 bytes each from shared memory, the copies write them once
  const double shared = (24.0 * (FF_BM + bn) * 32 + 3.0 * (FF_BM + bn / cg) * 128) / 120;
  const double main = (double)k64 * (S == 3 ? shared : (mul > fetch ? mul : fetch));
  // three planes, by width 64 / 128 / 256
  static const double epi3[3][3] = {{3000, 4000, 15500}, {12000, 15500, 48000}, {6000, 10000, 19000}};
  const double epi = S == 3 ? epi3[kind][bn == 64 ? 0 : (bn == 128 ? 1 : 2)] : bn * (kind == FF_DGATE ? 70.0 : 45.0);
  return S == 3 ? main + epi : (main > epi ? main : epi);
}
static FfnPlan ffn_plan(int S, int kind, const FfnProduct* p, int n) {
  static const int shapes[4][2] = {{256, 2}, {128, 2}, {128, 1}, {64, 1}};
  FfnPlan best = {256, 2, {1, 1, 1}};
  double best_cost = 1e300;
  for (int i = 0; i < 4; ++i) {
    const int bn = shapes[i][0], cg = shapes[i][1], tm = FF_BM * cg, units = sm_count() / cg;
    bool low = true;
    double tiles[3], total = 0;
    for (int j = 0; j < n; ++j) {
      low = low && p[j].M <= FF_BM;
      tiles[j] = (double)((p[j].M + tm - 1) / tm) * p[j].m_parts * ((p[j].cols + bn - 1) / bn);
      total += tiles[j] * ffn_tile_cost(bn, cg, S, kind, p[j].k64);
    }
    if (low && cg == 2) continue;
    for (int most = 1; most <= (kind == FF_PLAIN ? 16 : 1); most += most < 4 ? 1 : (most < 8 ? 2 : 4)) {
      // slices: one product `most`; several: those whose tiles are longer than 1 / most of an SM's load are cut to that
      FfnPlan plan = {bn, cg, {1, 1, 1}};
      double load = 0, largest = 0, join = 0;
      bool cut = false;
      for (int j = 0; j < n; ++j) {
        long long q = most;
        if (n > 1) q = (long long)(ffn_tile_cost(bn, cg, S, kind, p[j].k64) * units * most / total);
        if (q > p[j].k64 / 4) q = p[j].k64 / 4;
        if (q > 16) q = 16;
        if (most == 1 || q < 1 || (long long)p[j].m_parts * ((p[j].M + 31) / 32) > 65535) q = 1;      // 65535: grid of ffn_join_kernel
        plan.splits[j] = (int)q;
        const double c = ffn_tile_cost(bn, cg, S, kind, (p[j].k64 + q - 1) / q);
        load += tiles[j] * q * c;
        if (c > largest) largest = c;
        if (q > 1) {
          cut = true;
          join += 5000.0 + 8.0 * q * p[j].m_parts * p[j].M * p[j].cols / (30.0 * sm_count());
        }
      }
      if (most > 1 && !cut) continue;
      double cost = join + 3000.0;                       // launch, first loads
      if (n == 1) cost += largest * (double)(long long)((tiles[0] * plan.splits[0] + units - 1) / units);
      else cost += load / units + 0.5 * largest;
      if (cost < best_cost) { best_cost = cost; best = plan; }
    }
  }
  return best;
}
template <int S, int KIND>
static int ffn_launch(const FfnPlan& t, FfnBatch& batch, const FfnOperands* o, cudaStream_t st) {
  if (t.cg == 2) return t.bn == 256 ? ffn_launch_t<256, S, KIND, 2>(batch, o, st) : ffn_launch_t<128, S, KIND, 2>(batch, o, st);
  return t.bn == 128 ? ffn_launch_t<128, S, KIND, 1>(batch, o, st) : ffn_launch_t<64, S, KIND, 1>(batch, o, st);
}

static long long ffn_plane(int M, int N) { return (long long)((M + 31) / 32 * 32) * ((N + 15) / 16 * 16); }
static int ffn_k_blocks(int S, int k) { return (k + FF_BK(S) - 1) / FF_BK(S); }
static FfnProduct ffn_product(int S, int M, int m_parts, int cols, int k, int segments) {
  return {M, m_parts, cols, ((long long)ffn_k_blocks(S, k) * segments * FF_BK(S) + 63) / 64};
}
// floats of partial sums that plain products need
static long long ffn_partial_floats(const FfnPlan& plan, const FfnProduct* p, int n) {
  long long floats = 0;
  for (int j = 0; j < n; ++j)
    if (plan.splits[j] > 1) floats += plan.splits[j] * p[j].m_parts * ffn_plane(p[j].M, p[j].cols);
  return floats;
}
// the products of the two plain launches: Y;  dX, dW_in, dW_out
static FfnProduct ffn_y_product(int S, int m, int f, int n) { return ffn_product(S, m, 1, n, f, 1); }
static void ffn_grad_products(int S, int m, int d, int f, int n, FfnProduct (&p)[3]) {
  p[0] = ffn_product(S, m, 1, d, f, 2);
  p[1] = ffn_product(S, f, 2, d, m, 1);
  p[2] = ffn_product(S, n, 1, f, m, 1);
}

// gate, dgate
template <int KIND>
static int ffn_gemm(int S, const FfnGemm& g, const FfnOperand& a, const FfnOperand& b, int k, cudaStream_t st) {
  const FfnProduct p = ffn_product(S, g.M, 1, KIND == FF_GATE ? 2 * g.N : g.N, k, 1);
  const FfnPlan plan = ffn_plan(S, KIND, &p, 1);
  FfnBatch batch = {};
  batch.g[0] = g;
  batch.g[0].k_splits = 1;
  batch.n = 1;
  const FfnOperands o = {a, b};
  return S == 3 ? ffn_launch<3, KIND>(plan, batch, &o, st) : ffn_launch<1, KIND>(plan, batch, &o, st);
}
// plain products of S operand planes, g[i].out [m_parts M, N]; partial: scratch of ffn_partial_floats
static int ffn_plain(int S, const FfnPlan& plan, FfnBatch& batch, const int* index, const FfnOperands* o, int dt, float* partial,
                     cudaStream_t st) {
  for (int i = 0; i < batch.n; ++i) {
    FfnGemm& g = batch.g[i];
    g.ldo = g.N;
    g.vec16 = (((uintptr_t)g.out | (uintptr_t)((long long)g.N * dt_bytes(dt))) & 15) == 0;
    g.k_splits = plan.splits[index[i]];
    if (g.k_splits == 1) continue;
    if (partial == nullptr) return -1;
    g.z = partial;
    g.ldz = (g.N + 15) / 16 * 16;
    g.z_plane = ffn_plane(g.M, g.N);
    partial += g.k_splits * g.m_parts * g.z_plane;
  }
  int rc = S == 3 ? ffn_launch<3, FF_PLAIN>(plan, batch, o, st) : ffn_launch<1, FF_PLAIN>(plan, batch, o, st);
  for (int i = 0; i < batch.n && !rc; ++i) {
    const FfnGemm& g = batch.g[i];
    if (g.k_splits == 1) continue;
    const dim3 grid((g.N + 63) / 64, g.m_parts * ((g.M + 31) / 32)), block(256);
    if (dt == DT_F32)
      rc = (int)launch_k_if(ffn_chain.dependent(), ffn_join_kernel<float>, grid, block, 0, st, (const float*)g.z, g.ldz, g.z_plane, g.k_splits, g.m_parts,
                         g.M, g.N, (float*)g.out);
    else if (dt == DT_BF16)
      rc = (int)launch_k_if(ffn_chain.dependent(), ffn_join_kernel<__nv_bfloat16>, grid, block, 0, st, (const float*)g.z, g.ldz, g.z_plane, g.k_splits,
                         g.m_parts, g.M, g.N, (__nv_bfloat16*)g.out);
    else
      rc = (int)launch_k_if(ffn_chain.dependent(), ffn_join_kernel<__half>, grid, block, 0, st, (const float*)g.z, g.ldz, g.z_plane, g.k_splits, g.m_parts,
                         g.M, g.N, (__half*)g.out);
  }
  return rc;
}

// A matrix the products can read: itself, or its image `dst` in the workspace, which `images` then has to make (src null:
// the image is there already)
static void ffn_prepare(FfnOperand* o, const void* src, long long rows, int cols, long long ld, int parts, int dt, void* dst,
                        FfnImages* images) {
  o->rows = (int)(rows / parts);
  o->cols = cols;
  o->parts = parts;
  o->splits = dt == DT_F32 ? 3 : 1;
  o->p = dst == nullptr ? src : dst;
  o->ld = dst == nullptr ? ld : pad16(cols);
  if (dst == nullptr || src == nullptr) return;
  FfnImage& m = images->m[images->n++];
  const uintptr_t bits = (uintptr_t)src | (uintptr_t)(ld * dt_bytes(dt));
  m.src = src; m.dst = reinterpret_cast<uint16_t*>(dst); m.rows = rows; m.lds = ld; m.cols = cols; m.ldd = pad16(cols);
  m.vec = bits % (4 * dt_bytes(dt)) == 0 ? 4 : (bits % (2 * dt_bytes(dt)) == 0 ? 2 : 1);
}
static int ffn_make_images(FfnImages& images, int dt, cudaStream_t st) {
  if (images.n == 0) return 0;
  long long blocks = 0;
  for (int k = 0; k < images.n; ++k) {
    const long long runs = images.m[k].rows * (images.m[k].ldd / 8);
    images.m[k].first_block = (unsigned)blocks;
    blocks += (runs + 255) / 256;
    if (runs > 0xffffff00LL || blocks > 0x7fffffffLL) return -1;
  }
  const dim3 grid((unsigned)blocks), block(256);
  return (int)(dt == DT_F32 ? launch_k_if(ffn_chain.dependent(), ffn_operand_kernel<3>, grid, block, 0, st, images)
                            : launch_k_if(ffn_chain.dependent(), ffn_operand_kernel<1>, grid, block, 0, st, images));
}

struct FfnShape {
  int m, d, f, n, act, dt;
};
static bool ffn_shape_ok(const FfnShape& s) {
  const long long big = 0x7fffff00LL;
  return s.m > 0 && s.d > 0 && s.f > 0 && s.n > 0 && s.dt >= 0 && s.dt <= 2 && s.act >= 0 && s.act <= 3 &&
         s.m < big && s.d < big && 2LL * s.f < big && s.n < big;
}
// floats of the scratch `partial` of either pass (0: none)
extern "C" long long gated_ffn_partial_floats(int m, int d, int f, int n, int dt, int backward) {
  const int S = dt == DT_F32 ? 3 : 1;
  if (m <= 0 || d <= 0 || f <= 0 || n <= 0) return 0;
  FfnProduct p[3];
  if (backward) ffn_grad_products(S, m, d, f, n, p);
  else p[0] = ffn_y_product(S, m, f, n);
  return ffn_partial_floats(ffn_plan(S, FF_PLAIN, p, backward ? 3 : 1), p, backward ? 3 : 1);
}

// The tiles that a training pass runs with, for tests: launches gate, Y, dgate, gradients x (accumulator columns, CTAs per tile,
// slices of k of up to three products)
extern "C" void gated_ffn_plan(int m, int d, int f, int n, int dt, int* out) {
  const int S = dt == DT_F32 ? 3 : 1;
  FfnProduct p[3];
  FfnPlan plan[4];
  p[0] = ffn_product(S, m, 1, 2 * f, d, 1);
  plan[0] = ffn_plan(S, FF_GATE, p, 1);
  p[0] = ffn_y_product(S, m, f, n);
  plan[1] = ffn_plan(S, FF_PLAIN, p, 1);
  p[0] = ffn_product(S, m, 1, f, n, 1);
  plan[2] = ffn_plan(S, FF_DGATE, p, 1);
  ffn_grad_products(S, m, d, f, n, p);
  plan[3] = ffn_plan(S, FF_PLAIN, p, 3);
  for (int i = 0; i < 4; ++i) {
    out[5 * i] = plan[i].bn;
    out[5 * i + 1] = plan[i].cg;
    for (int j = 0; j < 3; ++j) out[5 * i + 2 + j] = plan[i].splits[j];
  }
}

// whether an evaluation pass takes the form for few tokens (`few` of gated_ffn_forward)
extern "C" int gated_ffn_few(int m, int d, int f, int n, int dt) { return ffn_few_fits(m, d, f, n, dt); }

static int ffn_forward(const FfnForwardCall* c) {
  const void *x = c->x, *w_in = c->w_in, *w_out = c->w_out;
  void *x_img = c->x_img, *in_img = c->in_img, *out_img = c->out_img, *h = c->h, *y = c->y;
  float *z = c->z, *partial = c->partial;
  const long long ldx = c->ldx, ld_in = c->ld_in, ld_out = c->ld_out;
  const int m = (int)c->m, d = (int)c->d, f = (int)c->f, n = (int)c->n, act = (int)c->act, dt = (int)c->dt;
  const cudaStream_t st = (cudaStream_t)c->st;
  const FfnShape s = {m, d, f, n, act, dt};
  ffn_chain = FfnChain();
  if (!ffn_shape_ok(s)) return -1;
  if (c->few) {
    ffn_chain.launches = 2;
    return ffn_few_forward(x, ldx, w_in, ld_in, w_out, ld_out, reinterpret_cast<float*>(h), y, m, d, f, n, act, dt, st);
  }
  FfnOperand ox, oi, oo;
  FfnImages images = {};
  ffn_prepare(&ox, x, m, d, ldx, 1, dt, x_img, &images);
  ffn_prepare(&oi, w_in, 2LL * f, d, ld_in, 2, dt, in_img, &images);
  ffn_prepare(&oo, w_out, n, f, ld_out, 1, dt, out_img, &images);
  int rc = ffn_make_images(images, dt, st);
  if (rc) return rc;
  const int S = dt == DT_F32 ? 3 : 1;
  FfnGemm g = {};
  g.fp16 = dt == DT_F16;
  g.act = act;
  g.segments = g.m_parts = g.a_parts = 1;
  g.b_parts = 2;
  g.M = m; g.N = f; g.k_blocks = ffn_k_blocks(S, d);
  g.out = h; g.ldo = pad16(f); g.vec16 = 1; g.z = z; g.ldz = pad16(f); g.z_plane = ffn_plane(m, f);
  rc = ffn_gemm<FF_GATE>(S, g, ox, oi, d, st);
  if (rc) return rc;
  const FfnOperands o = {{h, m, f, 1, S, pad16(f)}, oo};
  FfnBatch batch = {};
  batch.n = 1;
  FfnGemm& b = batch.g[0];
  b.fp16 = g.fp16;
  b.segments = b.m_parts = b.a_parts = b.b_parts = 1;
  b.M = m; b.N = n; b.k_blocks = ffn_k_blocks(S, f);
  b.out = y;
  const FfnProduct p = ffn_y_product(S, m, f, n);
  const int index = 0;
  return ffn_plain(S, ffn_plan(S, FF_PLAIN, &p, 1), batch, &index, &o, dt, partial, st);
}

static int ffn_backward(const FfnBackwardCall* c) {
  const void *x = c->x, *w_in = c->w_in, *w_out = c->w_out, *dy = c->dy, *h = c->h;
  void *x_img = c->x_img, *in_img = c->in_img, *out_img = c->out_img, *dy_img = c->dy_img, *dz = c->dz;
  void *dx = c->dx, *dw_in = c->dw_in, *dw_out = c->dw_out;
  float *z = c->z, *partial = c->partial;
  const long long ldx = c->ldx, ld_in = c->ld_in, ld_out = c->ld_out, ldy = c->ldy;
  const int m = (int)c->m, d = (int)c->d, f = (int)c->f, n = (int)c->n, act = (int)c->act, dt = (int)c->dt;
  const cudaStream_t st = (cudaStream_t)c->st;
  const FfnShape s = {m, d, f, n, act, dt};
  ffn_chain = FfnChain();
  if (!ffn_shape_ok(s)) return -1;
  const int S = dt == DT_F32 ? 3 : 1;
  FfnOperand ox, oi, oo, oy;
  FfnImages images = {};
  ffn_prepare(&oy, dy, m, n, ldy, 1, dt, dy_img, &images);
  ffn_prepare(&ox, x_img != nullptr && !(c->make & 1) ? nullptr : x, m, d, ldx, 1, dt, x_img, &images);
  ffn_prepare(&oi, in_img != nullptr && !(c->make & 2) ? nullptr : w_in, 2LL * f, d, ld_in, 2, dt, in_img, &images);
  ffn_prepare(&oo, out_img != nullptr && !(c->make & 4) ? nullptr : w_out, n, f, ld_out, 1, dt, out_img, &images);
  int rc = ffn_make_images(images, dt, st);
  if (rc) return rc;
  const FfnOperand oh = {h, m, f, 1, S, pad16(f)}, oz = {dz, m, f, 2, S, pad16(f)};
  FfnGemm base = {};
  base.fp16 = dt == DT_F16;
  base.act = act;
  base.segments = base.m_parts = base.a_parts = base.b_parts = 1;
  if (dx != nullptr || dw_in != nullptr) {
    FfnGemm g = base;
    g.M = m; g.N = f; g.k_blocks = ffn_k_blocks(S, n); g.b_mn = 1;
    g.out = dz; g.ldo = pad16(f); g.vec16 = 1; g.z = z; g.ldz = pad16(f); g.z_plane = ffn_plane(m, f);
    if ((rc = ffn_gemm<FF_DGATE>(S, g, oy, oo, n, st))) return rc;
  }
  // the plan is that of all three products whichever are wanted: a gradient's bits do not depend on the others
  FfnProduct p[3];
  ffn_grad_products(S, m, d, f, n, p);
  const FfnPlan plan = ffn_plan(S, FF_PLAIN, p, 3);
  FfnBatch batch = {};
  FfnOperands o[3];
  int index[3];
  if (dx != nullptr) {
    FfnGemm& g = batch.g[batch.n] = base;
    g.M = m; g.N = d; g.k_blocks = ffn_k_blocks(S, f); g.segments = 2; g.a_parts = g.b_parts = 2; g.b_mn = 1;
    g.out = dx;
    o[batch.n] = {oz, oi};
    index[batch.n++] = 0;
  }
  if (dw_in != nullptr) {
    FfnGemm& g = batch.g[batch.n] = base;
    g.M = f; g.N = d; g.k_blocks = ffn_k_blocks(S, m); g.m_parts = g.a_parts = 2; g.a_mn = g.b_mn = 1;
    g.out = dw_in;
    o[batch.n] = {oz, ox};
    index[batch.n++] = 1;
  }
  if (dw_out != nullptr) {
    FfnGemm& g = batch.g[batch.n] = base;
    g.M = n; g.N = f; g.k_blocks = ffn_k_blocks(S, m); g.a_mn = g.b_mn = 1;
    g.out = dw_out;
    o[batch.n] = {oy, oh};
    index[batch.n++] = 2;
  }
  return batch.n ? ffn_plain(S, plan, batch, index, o, dt, partial, st) : 0;
}

// whether launches inside a call are programmatic dependents in this process
extern "C" int choco_pdl_in_call() { return pdl_in_call() || pdl_enabled(); }

extern "C" int gated_ffn_forward(FfnForwardCall* c) {
  const int rc = ffn_forward(c);
  c->launches = ffn_chain.launches;
  return rc;
}
extern "C" int gated_ffn_backward(FfnBackwardCall* c) {
  const int rc = ffn_backward(c);
  c->launches = ffn_chain.launches;
  return rc;
}

// 0, or 1 after a bounded wait of a kernel on the current device ran out since the last call (synchronises)
extern "C" int gated_ffn_last_error() {
  int v = -1;
  if (cudaMemcpyFromSymbol(&v, g_ffn_error, sizeof(int)) != cudaSuccess) return -1;
  const int none = 0;
  if (v != 0) cudaMemcpyToSymbol(g_ffn_error, &none, sizeof(int));
  return v;
}
