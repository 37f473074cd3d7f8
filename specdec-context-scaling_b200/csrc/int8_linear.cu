// int8_linear.cu -- linear layer over 8-bit activations and weights:
//   y[r][n] = (sum_k a[r][k] w[n][k]) * a_scale[r] * w_scale[n] + bias[n]
// The integer sum is exact in any order: it lies in -2^31 < sum <= 2^31 for K <= 131072, whatever the codes.
// +2^31 itself (every product 128^2 at the largest K) converts to fp32 as 2^31 - 1 does: the tensor cores are
// told to saturate there, and where warps or CTAs add up it wraps to -2^31, which no other sum is (unwrapped).
// Scales and bias are applied in fp32 and the result is rounded once to the output type.
//
// Two kernels (few_rows):
//
// linear_int8_few_kernel, up to 8 rows, and up to 32 where that is ahead: bound by reading W once.
// Its comment is beside it.
//
// linear_int8_kernel, on the fifth-generation tensor cores, 320 threads.  The weight is the M operand:
// a tile is 128 output channels by up to 256 rows ("tokens") of a, so a call of few tokens wastes only
// columns of a narrow N, and an accumulator lane is an output channel.
//   warp 8    producer: TMA loads of the W tile [128 channels][128 codes] and the a tile
//             [tokens][128 codes] of each 128-code chunk of K (128-byte swizzle, K-major; the
//             ragged ends of K, N and the rows are filled with zeros by the TMA unit) into a
//             ring of 4 to 11 stages;
//   warp 9    one lane issues tcgen05.mma kind::i8 (K 32) into one of two TMEM accumulators,
//             so a tile's epilogue overlaps the next tile's products;
//   warps 0-7 epilogue: scales, bias, rounding and stores, two warps to a lane quarter.
// CG = 2: two CTAs on one 256-channel tile (cta_group::2).  Each loads its own 128 channels and
// half of the tokens, so a chunk costs a CTA 128 + tokens / 2 rows of loads where one CTA alone
// pays 128 + tokens; the pair's first CTA issues the products.  L2 delivers about 64 bytes a clock
// and SM, which a 256 x 256 pair needs exactly at the products' full rate: 8192^3 runs at 3.2-3.3
// POP/s, twice the bf16 rate of the library's product (3.29).  With K = 1536 and 17920 channels the
// output (1.2 GB for 32768 rows) shares L2 with those loads: 600-735 us, 2.5-3.0 POP/s, by the clock that the
// power cap leaves.
// splits > 1 (CG = 1): a cluster of `splits` CTAs shares one tile, each taking a share of the
// chunks of K and pushing its integer partial sums into the shared memory of the CTA that adds them up.
#include <cudaTypedefs.h>

#include <atomic>

#include "sd_common.cuh"
#include "sd_internal.h"
#include "umma.cuh"

namespace sd {

constexpr int kMaxWidth = 131072;
constexpr int kMaxRows = 1 << 21;
constexpr int kLinEpiWarps = 8;
constexpr int kLinThreads = 32 * (kLinEpiWarps + 2);
constexpr int kLinChunk = 128;                   // codes of K per stage
constexpr int kLinCh = 128;                      // channels per CTA
constexpr int kLinWTile = kLinCh * kLinChunk;    // 16 KB
constexpr int kLinMaxStages = 11;
constexpr int kLinRing = 204 * 1024;
constexpr int kLinMaxTokens = 256;
constexpr int kLinSplitTokens = 128;             // of a split tile: its partial sums take 512 bytes each

struct LinParams {
  const float* a_scale;
  const float* w_scale;
  const float* bias;
  void* out;
  int64_t out_stride;
  int32_t rows, n, chunks;
  int32_t tokens;    // tokens of a tile (the MMA's N)
  int32_t ch_tiles;  // tiles along the channels
  int32_t units;     // tiles of the call
  int32_t splits, stages, tmem_cols, weight_ready;
  int32_t vec_out;  // four outputs of a row can be stored at once
  int32_t rows16;   // rows of the output are 16-byte aligned and whole 16-byte pieces
  int32_t* status;
  uint64_t wait_ns;  // limit of a wait
};

// ---------------------------------------------------------------- PTX of this kernel
// instruction descriptor of kind::i8: signed x signed -> s32, both operands K-major
SD_DEV uint32_t idesc_i8(int M, int N, bool saturate) {
  return (saturate ? 1u << 3 : 0u) | (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}
// One lane of a converged warp.  The loops around it stay warp-uniform, so descriptors, barriers and
// loop counters live in uniform registers (the tcgen05 operands): a loop inside `if (lane == 0)`
// moved every operand there first, and cost 6 % of the whole at 8192^3 (398 and 375 us).
SD_DEV bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(p));
  return p != 0;
}
template <int CG>
SD_DEV void mma_i8_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  const uint32_t acc = accumulate ? 1u : 0u;
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
}
// arrive on `bar` (of both CTAs of a pair) when the MMAs issued so far are complete
template <int CG>
SD_DEV void commit_mma(uint64_t* bar) {
  if constexpr (CG == 1)
    umma::commit(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}
template <int CG>
SD_DEV void tmem_alloc_cg(uint32_t* result, uint32_t ncols) {
  if constexpr (CG == 1) {
    umma::tmem_alloc(result, ncols);
    umma::tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(result)),
                 "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
  }
}
template <int CG>
SD_DEV void tmem_dealloc_cg(uint32_t taddr, uint32_t ncols) {
  if constexpr (CG == 1)
    umma::tmem_dealloc(taddr, ncols);
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// 2-D tile load; CG = 2: `bar` may be the barrier of the pair's other CTA
template <int CG>
SD_DEV void tma_codes(void* dst, const CUtensorMap* map, int32_t k, int32_t row, uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(k), "r"(row), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(k), "r"(row), "r"(bar)
        : "memory");
}
// Arrive on a barrier of another CTA of the cluster (or on one's own, by its cluster address).  It
// hands back an accumulator whose reads are complete (tcgen05.wait::ld), no memory: a release at
// cluster scope would first wait for all of the warp's output stores.
SD_DEV void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The same with a release: what this thread wrote, or saw written before a barrier, to that CTA is there.
SD_DEV void mbar_arrive_release_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
SD_DEV void dsmem_st_s32(uint32_t addr, int32_t v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
// warp_wait that also acquires what other CTAs of the cluster released
SD_DEV bool warp_wait_cluster(uint64_t* bar, uint32_t parity) {
  const bool ok = warp_wait(bar, parity);
  asm volatile("fence.acq_rel.cluster;" ::: "memory");
  return ok;
}
SD_DEV void tmem_ld16_s32(uint32_t ta, int32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(ta));
}
// wait for this thread's TMEM loads; `v` may be used from here on
SD_DEV void tmem_wait_ld16(int32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])::"memory");
}
// 32 lanes x 16 columns as two halves of 16 lanes (16x256b): v[8 h + 4 j + 2 q + e] is lane
// 16 h + 8 q + T / 4, column 8 j + 2 (T % 4) + e of thread T -- the fragments of 8 x 8 matrices that
// stmatrix takes
SD_DEV void tmem_ld_fragments(uint32_t ta, int32_t (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(ta));
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(ta + (16u << 16)));
}
// four 8 x 8 matrices of 16-bit values, stored transposed: lane 8 i + k gives the address of column k of
// matrix i
SD_DEV void stmatrix_trans(uint32_t addr, uint32_t m0, uint32_t m1, uint32_t m2, uint32_t m3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(m0), "r"(m1),
               "r"(m2), "r"(m3)
               : "memory");
}
template <typename T>
SD_DEV void store_out(T* p, float v) {
  if constexpr (sizeof(T) == 4)
    *p = v;
  else
    *p = __float2bfloat16_rn(v);
}
// NaN for this lane's channel of tokens c0 .. c1 - 1: of a tile whose products did not come
template <typename T>
SD_DEV void store_lost(T* o, int64_t stride, int c0, int c1) {
  for (int c = c0; c < c1; ++c) store_out(o + c * stride, __int_as_float(0x7FC00000));
}
// A sum whose conversion to fp32 is that of the sum without wrapping: +2^31, wrapped to -2^31, becomes 2^31 - 1,
// which converts to 2^31.
SD_DEV int32_t unwrapped(int32_t sum) { return sum == INT32_MIN ? INT32_MAX : sum; }
SD_DEV float scaled(int32_t acc, float sa, float sw, float b) {
  return __fmaf_rn(__fmul_rn(static_cast<float>(acc), sa), sw, b);
}

// 16 tokens of one channel (lane = channel, any alignment, f32 or bf16): scaled, rounded, stored, 32
// neighbouring channels of a token at a time.  All scales are read and all results formed before the
// first store, so nothing waits behind a store (one by one: 1.9 times the time at 32768 x 1536 x 17920).
template <typename T, bool GUARD>
SD_DEV void store_tokens(const int32_t (&v)[16], const float* s_scale, float sw, float bias, T* o, int64_t stride,
                         int ntok) {
  float sa[16];
#pragma unroll
  for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(sa + i) = *reinterpret_cast<const float4*>(s_scale + i);
  float y[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i] = scaled(v[i], sa[i], sw, bias);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (!GUARD || i < ntok) store_out(o, y[i]);
    o += stride;
  }
}

// two fp32 products / sums at once (sm_100's packed arithmetic; each is the scalar operation's result)
SD_DEV uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
SD_DEV uint32_t scaled_pair(int32_t a0, int32_t a1, uint64_t sa, uint64_t sw, uint64_t bias) {
  uint64_t y = pair_of(static_cast<float>(a0), static_cast<float>(a1));
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(y) : "l"(sa));
  asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(y) : "l"(sw), "l"(bias));
  float lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(y));
  return pack_bf16(lo, hi);
}

// bf16 results of 32 channels x 16 tokens, held as fragments, to 64 consecutive bytes of each token's row
// by way of 1 KB of shared memory: eight tokens a store instead of half of one.  `put`: this lane's
// address for stmatrix, `get`: for reading back; o: this lane's 16 bytes of tokens lane / 4 and, `half`
// further, lane / 4 + 8.  At short K the epilogue bounds the kernel: with one 2-byte store a token and
// a tile's scales loaded at its start, 8192 x 896 x 9728 took 72 us; so, 60 to 65.
template <bool GUARD>
SD_DEV void store_fragments(const int32_t (&v)[16], const float* s_scale, const uint64_t (&sw)[4],
                            const uint64_t (&bias)[4], uint32_t put, const uint8_t* get, uint8_t* o, int64_t half,
                            int ntok, bool ch_ok) {
  const int lane = threadIdx.x & 31, t = lane & 3;
  const uint64_t sa[2] = {*reinterpret_cast<const uint64_t*>(s_scale + 2 * t),
                          *reinterpret_cast<const uint64_t*>(s_scale + 8 + 2 * t)};
  __syncwarp();  // the stage's previous contents are read
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t m[4];  // (tokens 0-7, channels 0-7), (tokens 0-7, channels 8-15), then tokens 8-15
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 2; ++q)
        m[2 * j + q] = scaled_pair(v[8 * h + 4 * j + 2 * q], v[8 * h + 4 * j + 2 * q + 1], sa[j], sw[2 * h + q],
                                   bias[2 * h + q]);
    stmatrix_trans(put ^ (h * 32u), m[0], m[1], m[2], m[3]);
  }
  __syncwarp();
  const uint4 r0 = *reinterpret_cast<const uint4*>(get), r1 = *reinterpret_cast<const uint4*>(get + 512);
  if (!GUARD || (ch_ok && (lane >> 2) < ntok)) *reinterpret_cast<uint4*>(o) = r0;
  if (!GUARD || (ch_ok && (lane >> 2) + 8 < ntok)) *reinterpret_cast<uint4*>(o + half) = r1;
}

// A split tile: the CTAs of the cluster have pushed their partial sums of this CTA's tokens (every
// `splits`-th, from `rank` on) into `got` [split][token][128 channels]; a warp adds up a token, a lane four
// channels.  `lost`: sums are missing, the results are NaN.
template <typename T>
SD_DEV void add_partials(const LinParams& p, const int32_t* got, int rank, int unit, bool lost) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, share = p.tokens / p.splits;
  const int tt = unit / p.ch_tiles, ct = unit - tt * p.ch_tiles;
  const int n = ct * kLinCh + lane * 4;
  const int tok0 = tt * p.tokens, ntok = min(p.tokens, p.rows - tok0);
  float sw[4] = {}, bias[4] = {};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (n + j < p.n) {
      sw[j] = p.w_scale[n + j];
      if (p.bias) bias[j] = p.bias[n + j];
    }
  for (int i = warp; i < share; i += kLinEpiWarps) {
    const int c = rank + p.splits * i;
    if (c >= ntok) break;
    const float sa = lost ? __int_as_float(0x7FC00000) : p.a_scale[tok0 + c];
    uint4 sum = make_uint4(0, 0, 0, 0);
#pragma unroll 8
    for (int r = 0; r < p.splits; ++r) {
      const uint4 v = *reinterpret_cast<const uint4*>(got + (r * share + i) * kLinCh + lane * 4);
      sum.x += v.x;
      sum.y += v.y;
      sum.z += v.z;
      sum.w += v.w;
    }
    const float y[4] = {scaled(unwrapped(sum.x), sa, sw[0], bias[0]), scaled(unwrapped(sum.y), sa, sw[1], bias[1]),
                        scaled(unwrapped(sum.z), sa, sw[2], bias[2]), scaled(unwrapped(sum.w), sa, sw[3], bias[3])};
    T* o = static_cast<T*>(p.out) + (tok0 + c) * p.out_stride + n;
    if (p.vec_out && n + 4 <= p.n) {
      if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(o) = make_float4(y[0], y[1], y[2], y[3]);
      else
        *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < p.n) store_out(o + j, y[j]);
    }
  }
}

// ---------------------------------------------------------------- the kernel
template <int CG, typename T>
__global__ void __launch_bounds__(kLinThreads, 1)
    linear_int8_kernel(const LinParams p, const __grid_constant__ CUtensorMap amap,
                       const __grid_constant__ CUtensorMap wmap) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kLinMaxStages], empty[kLinMaxStages], acc_full[2], acc_empty[2], given_up, partials;
  __shared__ uint32_t tmem_base;
  __shared__ int32_t lost;  // splits: partial sums of the tile, of whichever CTA, did not come
  __shared__ __align__(16) float s_scale[kLinEpiWarps][kLinMaxTokens / 2];
  __shared__ __align__(128) uint8_t s_stage[kLinEpiWarps][1024];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int csize = CG == 2 ? 2 : p.splits;
  const int rank = csize > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit0 = blockIdx.x / csize, unit_step = gridDim.x / csize;
  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kLinEpiWarps * CG);
    }
    mbar_init(&given_up, 1);
    mbar_init(&partials, csize);
    lost = 0;
    fence_barrier_init();
  }
  if (warp == kLinEpiWarps && lane == 0) {
    prefetch_tmap(&amap);
    prefetch_tmap(&wmap);
  }
  if (warp == kLinEpiWarps + 1) tmem_alloc_cg<CG>(&tmem_base, p.tmem_cols);
  umma::fence_before_sync();
  __syncwarp();
  if (CG == 2) {
    cluster_sync();  // the partner's barriers are signalled from here on
  } else {
    if (csize > 1) cluster_arrive();  // partial sums are pushed once every CTA of the cluster is here
    __syncthreads();
  }
  umma::fence_after_sync();
  const uint32_t tbase = tmem_base;
  const int a_rows = p.tokens / CG;  // rows of a this CTA loads
  const int stage_bytes = kLinWTile + a_rows * kLinChunk;
  // this CTA's share of the chunks of K
  const int k_begin = CG == 2 ? 0 : static_cast<int>(static_cast<int64_t>(p.chunks) * rank / csize);
  const int k_end = CG == 2 ? p.chunks : static_cast<int>(static_cast<int64_t>(p.chunks) * (rank + 1) / csize);

  if (warp == kLinEpiWarps) {
    // ---- producer
    int s = 0;              // next stage to fill, and the parity of its last use's end
    uint32_t parity = 1;    // (a fresh barrier reads as "phase 1 is over")
    bool stop = false;
    bool waited = false;
    for (int u = unit0; u < p.units && !stop; u += unit_step) {
      const int tt = u / p.ch_tiles, ct = u - tt * p.ch_tiles;
      const int ch0 = (ct * CG + (CG == 2 ? rank : 0)) * kLinCh;
      const int tok0 = tt * p.tokens + (CG == 2 ? rank * a_rows : 0);
      int k = k_begin;
      if (!waited) {
        // the first stages' weights go out before the preceding kernel is over, if they may
        const int ahead = min(p.stages, k_end - k_begin);
        if (elect_one()) {
          if (!p.weight_ready) grid_dep_wait();
          for (int i = 0; i < ahead; ++i) {
            const uint32_t bar = CG == 2 ? dsmem_addr(smem_u32(&full[i]), 0) : smem_u32(&full[i]);
            if (CG == 1 || rank == 0) mbar_arrive_expect_tx(&full[i], CG * stage_bytes);
            tma_codes<CG>(smem + i * stage_bytes, &wmap, (k + i) * kLinChunk, ch0, bar);
          }
          if (p.weight_ready) grid_dep_wait();
          grid_dep_launch();
          for (int i = 0; i < ahead; ++i) {
            const uint32_t bar = CG == 2 ? dsmem_addr(smem_u32(&full[i]), 0) : smem_u32(&full[i]);
            tma_codes<CG>(smem + i * stage_bytes + kLinWTile, &amap, (k + i) * kLinChunk, tok0, bar);
          }
        }
        __syncwarp();
        k += ahead;
        s = ahead;
        if (s == p.stages) s = 0, parity = 0;
        waited = true;
      }
      for (; k < k_end; ++k) {
        if (!warp_wait(&empty[s], parity, p.wait_ns)) {
          if (lane == 0) raise_status(p.status, SPECDEC_STATUS_TIMEOUT);
          stop = true;
          break;
        }
        if (elect_one()) {
          uint8_t* st = smem + s * stage_bytes;
          const uint32_t bar = CG == 2 ? dsmem_addr(smem_u32(&full[s]), 0) : smem_u32(&full[s]);
          if (CG == 1 || rank == 0) mbar_arrive_expect_tx(&full[s], CG * stage_bytes);
          tma_codes<CG>(st, &wmap, k * kLinChunk, ch0, bar);
          tma_codes<CG>(st + kLinWTile, &amap, k * kLinChunk, tok0, bar);
        }
        __syncwarp();
        if (++s == p.stages) s = 0, parity ^= 1;
      }
    }
    // every stage's last use is over before the CTA leaves (bounded; unused stages pass at once) ...
    for (int i = 0, at = s; i < p.stages && !stop; ++i, at = at + 1 == p.stages ? 0 : at + 1)
      stop = !warp_wait(&empty[at], at < s ? parity ^ 1 : parity);
    // ... or, after a wait that gave up, at least the copies under way have landed (the first such wait that runs
    // out, for a stage that the pair's other CTA did not fill, has left time enough for all)
    for (int i = 0; i < p.stages && stop && (CG == 1 || rank == 0); ++i)
      if (!warp_wait(&full[i], i < s ? parity ^ 1 : parity)) break;
    if (CG == 1 && csize > 1) cluster_wait();
  } else if (warp == kLinEpiWarps + 1) {
    // ---- MMA issuer
    if (rank % CG == 0) {
      grid_dep_wait();  // a is loaded after the preceding kernel is over: the limit of the first wait starts here, too
      const uint32_t idesc = idesc_i8(kLinCh * CG, p.tokens, p.chunks == kMaxWidth / kLinChunk);
      const uint32_t ring = smem_u32(smem);
      int s = 0, ui = 0;
      uint32_t parity = 0;
      bool ok = true;
      bool ready = false;  // stage s was seen full already
      for (int u = unit0; u < p.units && ok; u += unit_step, ++ui) {
        const int b = ui & 1;
        // accumulator b is free once the epilogue has read unit ui - 2
        if (ui >= 2 && !warp_wait(&acc_empty[b], ((ui >> 1) - 1) & 1, p.wait_ns)) {
          ok = false;
          break;
        }
        umma::fence_after_sync();
        const uint32_t d = umma::taddr(tbase, 0, b * (p.tmem_cols / 2));
        for (int k = k_begin; k < k_end; ++k) {
          if (!__all_sync(0xffffffffu, ready) && !warp_wait(&full[s], parity, p.wait_ns)) {
            ok = false;
            break;
          }
          umma::fence_after_sync();
          // the next stage's barrier is read while this stage's products are issued
          const int s1 = s + 1 == p.stages ? 0 : s + 1;
          const uint32_t parity1 = s1 == 0 ? parity ^ 1 : parity;
          ready = mbar_test(&full[s1], parity1);
          // 32 codes further along K are 32 bytes, 2 in the descriptor's address field
          const uint64_t wd = umma::desc_kmajor_sw128(ring + s * stage_bytes);
          const uint64_t ad = umma::desc_kmajor_sw128(ring + s * stage_bytes + kLinWTile);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_i8_ss<CG>(d, wd + 2 * kk, ad + 2 * kk, idesc, k > k_begin || kk > 0);
            commit_mma<CG>(&empty[s]);
            if (k + 1 == k_end) commit_mma<CG>(&acc_full[b]);
          }
          s = s1;
          parity = parity1;
        }
      }
      if (!ok) {  // the products issued so far end before TMEM is given back
        if (elect_one()) {
          raise_status(p.status, SPECDEC_STATUS_TIMEOUT);
          commit_mma<CG>(&given_up);
        }
        __syncwarp();
        (void)warp_wait(&given_up, 0);
      }
    }
    __syncwarp();
    if (CG == 1 && csize > 1) cluster_wait();
  } else {
    // ---- epilogue: lane = channel, columns = tokens; two warps share a lane quarter, each half the tokens
    grid_dep_wait();
    T* out = static_cast<T*>(p.out);
    const int quarter = warp & 3, batches = p.tokens / 16;
    const int c0 = (warp >> 2) * (batches / 2) * 16, c1 = warp >= 4 ? p.tokens : batches / 2 * 16;
    // fragments: this thread's channels are T / 4 + {0, 8, 16, 24} of the quarter's, else lane T's
    const bool fragments = sizeof(T) == 2 && p.rows16;
    // lane 8 i + k of stmatrix stores token 8 (i / 2) + k, 16-byte chunk i % 2 (+ 2 in the second half) of its
    // 64 bytes, at chunk c ^ (token / 2 % 4): no bank conflicts either way
    const int put_token = (lane >> 4) * 8 + (lane & 7);
    const uint32_t put = smem_u32(s_stage[warp]) + put_token * 64 + ((((lane >> 3) & 1) ^ ((put_token >> 1) & 3)) << 4);
    const uint8_t* get = s_stage[warp] + (lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) << 4);
    int tt = unit0 / p.ch_tiles, ct = unit0 - tt * p.ch_tiles;
    const int step_tt = unit_step / p.ch_tiles, step_ct = unit_step - step_tt * p.ch_tiles;
    // a tile's scales are loaded while the tile before it is worked on, each channel's by one lane and shuffled to
    // its fragments (loaded by every lane that needs them: 62.9 and 58.8 us at 32768 x 64 x 4096)
    float sw_next = 0.f, bias_next = 0.f, sa_next[4];  // lane = channel, and tokens
    const auto load_scales = [&]() {
      const int nj = (ct * CG + (CG == 2 ? rank : 0)) * kLinCh + quarter * 32 + lane, t0 = tt * p.tokens + c0 + lane;
      const int t1 = min(tt * p.tokens + c1, p.rows);
      sw_next = nj < p.n ? p.w_scale[nj] : 0.f;
      if (p.bias) bias_next = nj < p.n ? p.bias[nj] : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) sa_next[j] = t0 + 32 * j < t1 ? p.a_scale[t0 + 32 * j] : 0.f;
    };
    if (p.splits == 1 && unit0 < p.units) load_scales();
    int32_t* got = reinterpret_cast<int32_t*>(smem + p.stages * stage_bytes);  // splits: pushed partial sums
    if (CG == 1 && csize > 1) cluster_wait();
    int ui = 0;
    for (int u = unit0; u < p.units; u += unit_step, ++ui) {
      const int b = ui & 1;
      const int nq = (ct * CG + (CG == 2 ? rank : 0)) * kLinCh + quarter * 32, n = nq + lane;
      const int tok0 = tt * p.tokens, ntok = min(p.tokens, p.rows - tok0);
      const float sw0 = sw_next, bias0 = bias_next;
      uint64_t sw[4], bias[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float swj = __shfl_sync(0xffffffffu, sw0, (lane >> 2) + 8 * j);
        const float biasj = __shfl_sync(0xffffffffu, bias0, (lane >> 2) + 8 * j);
        sw[j] = pair_of(swj, swj);
        bias[j] = pair_of(biasj, biasj);
      }
      if (p.splits == 1) {
        __syncwarp();  // the previous tile's scales are read
#pragma unroll
        for (int j = 0; j < 4; ++j) s_scale[warp][lane + 32 * j] = sa_next[j];
        __syncwarp();
      }
      tt += step_tt;
      ct += step_ct;
      if (ct >= p.ch_tiles) ct -= p.ch_tiles, ++tt;
      if (p.splits == 1 && u + unit_step < p.units) load_scales();
      if (p.wait_ns == 0 || !warp_wait(&acc_full[b], (ui >> 1) & 1, p.wait_ns)) {
        if (lane == 0) raise_status(p.status, SPECDEC_STATUS_TIMEOUT);
        if (p.splits > 1) {
          lost = 1;
        } else {  // no output of this tile and of those after it is left as it was
          for (; u < p.units; u += unit_step) {
            const int t0 = u / p.ch_tiles * p.tokens;
            const int nl = (u % p.ch_tiles * CG + (CG == 2 ? rank : 0)) * kLinCh + quarter * 32 + lane;
            if (nl < p.n) store_lost(out + t0 * p.out_stride + nl, p.out_stride, c0, min(c1, p.rows - t0));
          }
        }
        break;
      }
      umma::fence_after_sync();
      const uint32_t ta = umma::taddr(tbase, quarter * 32, b * (p.tmem_cols / 2));
      const bool whole = c1 <= ntok && nq + 32 <= p.n;
      if (p.splits == 1 && fragments) {
        if constexpr (sizeof(T) == 2) {
          uint8_t* o = reinterpret_cast<uint8_t*>(out + (tok0 + c0 + (lane >> 2)) * p.out_stride + nq + 8 * (lane & 3));
          const int64_t half = 8 * p.out_stride * static_cast<int64_t>(sizeof(T));
          const bool ch_ok = nq + 8 * (lane & 3) < p.n;
          int32_t v[2][16];
          if (c0 < c1) tmem_ld_fragments(ta + c0, v[0]);
#pragma unroll 1
          for (int c = c0; c < c1; c += 32) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int cc = c + 16 * h;
              if (cc >= c1) break;
              tmem_wait_ld16(v[h]);
              // the next 16 columns are on their way while these are scaled and stored
              if (cc + 16 < c1) tmem_ld_fragments(ta + cc + 16, v[1 - h]);
              const float* sa = &s_scale[warp][cc - c0];
              if (whole)
                store_fragments<false>(v[h], sa, sw, bias, put, get, o, half, 16, true);
              else
                store_fragments<true>(v[h], sa, sw, bias, put, get, o, half, ntok - cc, ch_ok);
              o += 2 * half;
            }
          }
        }
      } else if (p.splits == 1) {
        T* o = out + (tok0 + c0) * p.out_stride + n;
        const int mine = n < p.n ? ntok : 0;  // tokens this lane stores
        int32_t v[2][16];
        if (c0 < c1) tmem_ld16_s32(ta + c0, v[0]);
#pragma unroll 1
        for (int c = c0; c < c1; c += 32) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int cc = c + 16 * h;
            if (cc >= c1) break;
            tmem_wait_ld16(v[h]);
            if (cc + 16 < c1) tmem_ld16_s32(ta + cc + 16, v[1 - h]);
            T* oc = o + (cc - c0) * p.out_stride;
            if (whole)
              store_tokens<T, false>(v[h], &s_scale[warp][cc - c0], sw0, bias0, oc, p.out_stride, 16);
            else
              store_tokens<T, true>(v[h], &s_scale[warp][cc - c0], sw0, bias0, oc, p.out_stride, mine - cc);
          }
        }
      } else {
        // token c goes to CTA c % splits, as its (c / splits)-th
        const int log2 = __ffs(p.splits) - 1, share = p.tokens >> log2;
        const uint32_t mine = smem_u32(got) + (rank * share * kLinCh + quarter * 32 + lane) * 4;
#pragma unroll 1
        for (int c = c0; c < c1; c += 16) {
          int32_t v[16];
          tmem_ld16_s32(ta + c, v);
          tmem_wait_ld16(v);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int to = (c + i) & (p.splits - 1), at = (c + i) >> log2;
            dsmem_st_s32(dsmem_addr(mine + at * (kLinCh * 4), to), v[i]);
          }
        }
      }
      umma::fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2)
          mbar_arrive_cluster(dsmem_addr(smem_u32(&acc_empty[b]), 0));
        else
          mbar_arrive(&acc_empty[b]);
      }
    }
    if (CG == 1 && csize > 1) {
      // this CTA's partial sums are out, whatever became of its waits; then those of the others are in
      named_bar_sync(1, 32 * kLinEpiWarps);
      if (threadIdx.x < csize) {
        if (lost) dsmem_st_s32(dsmem_addr(smem_u32(&lost), threadIdx.x), 1);
        mbar_arrive_release_cluster(dsmem_addr(smem_u32(&partials), threadIdx.x));
      }
      __syncwarp();
      // Twice the limit of the one wait that another CTA's push can stand behind, counted from this CTA's own
      // push: a CTA leaves only when nothing more is pushed to it.
      const bool in = warp_wait_cluster(&partials, 0) || warp_wait_cluster(&partials, 0);
      if (!in && lane == 0) raise_status(p.status, SPECDEC_STATUS_TIMEOUT);
      add_partials<T>(p, got, rank, unit0, !in || lost);
    }
  }

  umma::fence_before_sync();
  __syncwarp();
  if (CG == 2)
    cluster_sync();
  else
    __syncthreads();
  if (warp == kLinEpiWarps + 1) {
    umma::fence_after_sync();
    tmem_dealloc_cg<CG>(tbase, p.tmem_cols);
  }
}

// ---------------------------------------------------------------- a few rows
// A call of up to 32 rows is bound by reading W once and by the chain of latencies around that.  Here a
// block takes 16 output channels and its warps a share of K each, straight from global memory into
// mma.sync fragments: no ring, barriers or TMEM to set up, and a small enough block that the next kernel
// on the stream starts beside it.  5 x 1536 x 2048 takes 1.7 us (4.2 in the tcgen05 kernel); 5 x 1536 x
// 17920 4.7 us from L2, 6.1 from HBM (4.5 TB/s), where the waves of blocks over the SMs bound it.
// mma.sync m16n8k32 multiplies in any order of K, so a lane's 16 consecutive codes of a row are its
// fragments of two products: lane (g, t) holds codes 16 t .. 16 t + 15 of channels g and g + 8 and of
// token g in each step of 64 codes.  Channels and tokens past the end read as zero.
constexpr int kFewRows = 32;
constexpr int kFewCh = 16;
constexpr int kFewStep = 64;
constexpr int kFewAhead = 4;  // steps whose loads of a are under way together (of W: all of a warp's share, or 5 to 9 at a time)

struct FewParams {
  const int8_t* a;
  const int8_t* w;
  const float* a_scale;
  const float* w_scale;
  const float* bias;
  void* out;
  int64_t a_stride, w_stride, out_stride;
  int32_t rows, n, width, weight_ready;
};

// codes k .. k + 15 of a row of `width` (16-byte aligned); zero past its end
SD_DEV uint4 load_codes16(const int8_t* row, int k, int width) {
  if (k + 16 <= width) return *reinterpret_cast<const uint4*>(row + k);
  uint4 v = make_uint4(0, 0, 0, 0);
  if (k < width) {
    uint32_t* words = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 15; ++i)
      if (k + i < width) words[i / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(row[k + i])) << (8 * (i % 4));
  }
  return v;
}
SD_DEV void mma_m16n8k32(int32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Products of one step of 64 codes: this lane's codes of channels g and g + 8, and of token 8 b + g.
template <int NB>
SD_DEV void few_step(int32_t (&d)[NB][4], const uint4& c0, const uint4& c1, const uint4 (&x)[NB]) {
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    mma_m16n8k32(d[b], c0.x, c1.x, c0.y, c1.y, x[b].x, x[b].y);
    mma_m16n8k32(d[b], c0.z, c1.z, c0.w, c1.w, x[b].z, x[b].w);
  }
}
// The warps' partial sums of 16 channels meet in shared memory; the block's threads scale and store them.
template <int NB, int WARPS, typename T>
SD_DEV void few_finish(const FewParams& p, const int32_t (&d)[NB][4], int32_t (*part)[NB * 8][kFewCh + 1], int n0) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // accumulator: channels g (d0, d1) and g + 8 (d2, d3), tokens 2 t and 2 t + 1
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][b * 8 + 2 * t + (i & 1)][g + (i >> 1) * 8] = d[b][i];
  // this thread's first output's scales are on their way while the block meets
  const int row0 = threadIdx.x / kFewCh, n = n0 + threadIdx.x % kFewCh;
  const bool mine = row0 < NB * 8 && row0 < p.rows && n < p.n;
  const float sw = mine ? p.w_scale[n] : 0.f, bias = mine && p.bias ? p.bias[n] : 0.f;
  float sa = mine ? p.a_scale[row0] : 0.f;
  __syncthreads();
  for (int row = row0; row < NB * 8 && row < p.rows && n < p.n; row += 2 * WARPS) {
    uint32_t sum = 0;
#pragma unroll
    for (int j = 0; j < WARPS; ++j) sum += static_cast<uint32_t>(part[j][row][threadIdx.x % kFewCh]);
    if (row != row0) sa = p.a_scale[row];
    store_out(static_cast<T*>(p.out) + row * p.out_stride + n, scaled(unwrapped(sum), sa, sw, bias));
  }
}

// A warp's share of K is at most AHEAD steps: all its loads are under way at once, those of W before the
// preceding kernel is over if they may.
template <int NB, int WARPS, int AHEAD, typename T>
__global__ void __launch_bounds__(32 * WARPS, AHEAD <= 3 && NB == 1 ? 4 : 1) linear_int8_few_kernel(const FewParams p) {
  __shared__ int32_t part[WARPS][NB * 8][kFewCh + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kFewCh;
  const int steps = (p.width + kFewStep - 1) / kFewStep;
  const int s_begin = steps * warp / WARPS, s_end = steps * (warp + 1) / WARPS;
  // first code of step j of this lane (past the row's end: zeros)
  const auto code = [&](int j) { return s_begin + j < s_end ? (s_begin + j) * kFewStep + t * 16 : p.width; };
  const int8_t* w0 = p.w + static_cast<int64_t>(n0 + g) * p.w_stride;
  uint4 wa[AHEAD], wb[AHEAD], x[AHEAD][NB];
  if (!p.weight_ready) grid_dep_wait();
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    wa[j] = n0 + g < p.n ? load_codes16(w0, code(j), p.width) : make_uint4(0, 0, 0, 0);
    wb[j] = n0 + g + 8 < p.n ? load_codes16(w0 + 8 * p.w_stride, code(j), p.width) : make_uint4(0, 0, 0, 0);
  }
  if (p.weight_ready) grid_dep_wait();
  grid_dep_launch();
#pragma unroll
  for (int j = 0; j < AHEAD; ++j)
#pragma unroll
    for (int b = 0; b < NB; ++b)
      x[j][b] = b * 8 + g < p.rows ? load_codes16(p.a + static_cast<int64_t>(b * 8 + g) * p.a_stride, code(j), p.width)
                                   : make_uint4(0, 0, 0, 0);
  int32_t d[NB][4] = {};
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) few_step<NB>(d, wa[j], wb[j], x[j]);
  few_finish<NB, WARPS, T>(p, d, part, n0);
}

// The same for a longer K: a warp's share in turns of AHEAD steps.
template <int NB, int WARPS, int AHEAD, typename T>
__global__ void __launch_bounds__(32 * WARPS) linear_int8_few_long_kernel(const FewParams p) {
  __shared__ int32_t part[WARPS][NB * 8][kFewCh + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kFewCh;
  const int steps = (p.width + kFewStep - 1) / kFewStep;
  const int s_begin = steps * warp / WARPS, s_end = steps * (warp + 1) / WARPS;
  const int8_t* w0 = p.w + static_cast<int64_t>(n0 + g) * p.w_stride;
  const bool has0 = n0 + g < p.n, has1 = n0 + g + 8 < p.n;
  int32_t d[NB][4] = {};
  if (!p.weight_ready) grid_dep_wait();
  bool waited = !p.weight_ready;
  for (int s = s_begin; s < s_end || !waited; s += AHEAD) {
    const auto code = [&](int j) { return s + j < s_end ? (s + j) * kFewStep + t * 16 : p.width; };
    uint4 wa[AHEAD], wb[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      wa[j] = has0 ? load_codes16(w0, code(j), p.width) : make_uint4(0, 0, 0, 0);
      wb[j] = has1 ? load_codes16(w0 + 8 * p.w_stride, code(j), p.width) : make_uint4(0, 0, 0, 0);
    }
    if (!waited) grid_dep_wait();
    if (s == s_begin) grid_dep_launch();
    waited = true;
#pragma unroll
    for (int h = 0; h < AHEAD; h += kFewAhead) {
      uint4 x[kFewAhead][NB];
#pragma unroll
      for (int j = 0; j < kFewAhead && h + j < AHEAD; ++j)
#pragma unroll
        for (int b = 0; b < NB; ++b)
          x[j][b] = b * 8 + g < p.rows
                        ? load_codes16(p.a + static_cast<int64_t>(b * 8 + g) * p.a_stride, code(h + j), p.width)
                        : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < kFewAhead && h + j < AHEAD; ++j) few_step<NB>(d, wa[h + j], wb[h + j], x[j]);
    }
  }
  few_finish<NB, WARPS, T>(p, d, part, n0);
}

// ---------------------------------------------------------------- host
// What a function keeps between calls (an entry point's address, an attribute that was set, an occupancy) is the
// same whichever thread finds it out; atomics, because several may at once.
static int encode_codes(CUtensorMap* map, const void* base, int64_t width, int64_t rows, int64_t stride, int box_rows) {
  static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> known{nullptr};
  PFN_cuTensorMapEncodeTiled_v12000 fn = known.load(std::memory_order_relaxed);
  if (fn == nullptr) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) != cudaSuccess ||
        qres != cudaDriverEntryPointSuccess)
      return fail(SPECDEC_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    known.store(fn, std::memory_order_relaxed);
  }
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
  const cuuint32_t box[2] = {kLinChunk, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SPECDEC_ERR_INVALID, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  return SPECDEC_OK;
}

struct LinShape {
  int cg, tokens, splits;
};

// Clusters of `size` CTAs that the device holds at once (a GPC's SMs do not divide evenly: 148, 74, 33
// and 15 for 1, 2, 4 and 8 on a B200); asked once per device.
static int resident_clusters(int size, int dev, int sms);

// Launch shape by an estimate of the time of a call in ns.  A 128-code chunk of K costs a CTA the largest
// of its products (1.29 a token: 128 x 128 x 32 products in 64 clocks), what issuing its loads, waits and
// products takes (108, or 92 in a pair, and 0.43 a row loaded) and its share of L2's bandwidth (9.3 TB/s);
// the tiles of a CTA follow one another in waves, each hiding the previous one's epilogue (1.35 a token); a
// pair costs 155 more, a split the exchange of the partial sums.  The figures fit 3000 timings of 120 layer
// shapes (40 to 3500 rows): the chosen shape is within 2 % of the best one on average and 15 % at worst.
static LinShape pick_shape(int rows, int n, int chunks, int sms, int dev) {
  LinShape best = {1, 16, 1};
  double best_ns = 1e30;
  const auto consider = [&](int cg, int tokens, int splits) {
    const int64_t units = static_cast<int64_t>((n + cg * kLinCh - 1) / (cg * kLinCh)) * ((rows + tokens - 1) / tokens);
    const int slots = cg == 2 ? sms / 2 : splits > 1 ? resident_clusters(splits, dev, sms) : sms;
    if (splits > 1 && (units > slots || tokens > kLinSplitTokens)) return;
    const double waves = static_cast<double>((units + slots - 1) / slots);
    const double ctas = static_cast<double>(units < slots ? units : slots) * (cg == 2 ? 2 : splits);
    const double loaded = kLinCh + static_cast<double>(tokens / cg);
    double chunk = 1.29 * tokens;
    const double issue = (cg == 2 ? 92.0 : 108.0) + 0.43 * loaded;
    if (issue > chunk) chunk = issue;
    if (ctas * loaded * (kLinChunk / 9290.0) > chunk) chunk = ctas * loaded * (kLinChunk / 9290.0);
    const double tile = chunk * ((chunks + splits - 1) / splits), epilogue = 1.35 * tokens;
    double ns = waves * tile + epilogue + (epilogue > tile ? (waves - 1) * (epilogue - tile) : 0.0);
    if (splits > 1) ns += 858.0 + 5.1 * tokens + 50.0 * splits;
    if (cg == 2) ns += 155.0;
    if (ns < best_ns) best_ns = ns, best = {cg, tokens, splits};
  };
  for (int tokens = 16; tokens <= kLinMaxTokens; tokens += tokens < 32 ? 16 : 32) {
    for (int splits = 1; splits <= 8 && splits * 2 <= (splits == 1 ? 2 : chunks); splits *= 2) consider(1, tokens, splits);
    if (tokens % 32 == 0) consider(2, tokens, 1);
    if (tokens >= rows) break;
  }
  return best;
}

static int resident_clusters(int size, int dev, int sms) {
  static std::atomic<int> known[64][9];  // zeros: not asked yet
  int n = known[dev][size].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(size * sms));
    cfg.blockDim = dim3(kLinThreads);
    cfg.dynamicSmemBytes = kLinRing + 1024;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(size);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int got = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&got, linear_int8_kernel<1, __nv_bfloat16>, &cfg);
    if (e != cudaSuccess) (void)cudaGetLastError();
    n = e == cudaSuccess && got > 0 ? got : sms / (2 * size);
    known[dev][size].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <int CG, typename T>
static int allow_ring(int dev) {
  static std::atomic<bool> set[64];
  if (!set[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(linear_int8_kernel<CG, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               kLinRing + 1024);
    if (e != cudaSuccess) return fail(SPECDEC_ERR_CUDA, "linear_int8: %s", cudaGetErrorString(e));
    set[dev].store(true, std::memory_order_release);
  }
  return SPECDEC_OK;
}

template <int CG, typename T>
static int launch_linear(const LinParams& p, const CUtensorMap& amap, const CUtensorMap& wmap, int grid, int smem,
                         int dev, cudaStream_t st) {
  if (int rc = allow_ring<CG, T>(dev)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kLinThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int cluster = CG == 2 ? 2 : p.splits;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, linear_int8_kernel<CG, T>, p, amap, wmap);
  if (e != cudaSuccess) return fail(SPECDEC_ERR_CUDA, "linear_int8_kernel launch: %s", cudaGetErrorString(e));
  return after_launch("linear_int8_kernel");
}

// Up to 8 rows always (5 x 1536 x 17920: 4.7 us, 6.9 in the tcgen05 kernel).  With more, each block reads
// more of a, and the tcgen05 kernel is ahead once there are many blocks an SM or, past 16 rows, K is long
// (us here and there: 16 x 1536 x 4000 2.9 and 4.9, x 8000 5.0 and 5.0, 16 x 8960 x 1536 5.8 and 6.8;
// 32 x 1536 x 4000 3.5 and 4.9, x 8000 6.6 and 5.1, 32 x 4864 x 896 5.8 and 4.7).
static bool few_rows(int64_t rows, int width, int n) {
  const int per_sm = (n + kFewCh * device_sm_count() - 1) / (kFewCh * device_sm_count());  // blocks
  if (rows <= 8) return true;
  if (rows <= 16) return per_sm <= (width <= 2048 ? 3 : 1);
  return rows <= kFewRows && width <= 2048 && per_sm <= 2;
}
template <int NB, int WARPS, int AHEAD, typename T>
static int launch_few_as(const FewParams& p, cudaStream_t st) {
  return launch_pdl("linear_int8_few_kernel", linear_int8_few_kernel<NB, WARPS, AHEAD, T>,
                    dim3(static_cast<unsigned>((p.n + kFewCh - 1) / kFewCh)), dim3(32 * WARPS), 0, st, p);
}
template <int NB, int AHEAD, typename T>
static int launch_few_long(const FewParams& p, cudaStream_t st) {
  return launch_pdl("linear_int8_few_long_kernel", linear_int8_few_long_kernel<NB, 16, AHEAD, T>,
                    dim3(static_cast<unsigned>((p.n + kFewCh - 1) / kFewCh)), dim3(512), 0, st, p);
}
template <int NB, typename T>
static int launch_few(const FewParams& p, cudaStream_t st) {
  // a warp's share of K as far as registers let it be under way at once: 2 to 4 steps in a block of 8 warps
  // (K <= 2048), up to 5 or 9 in one of 16
  const int steps = (p.width + kFewStep - 1) / kFewStep;
  if (steps <= 16) return launch_few_as<NB, 8, 2, T>(p, st);
  if (steps <= 24) return launch_few_as<NB, 8, 3, T>(p, st);
  if (NB == 4 || steps <= 32) return launch_few_as<NB, 8, 4, T>(p, st);  // (few_rows: NB = 4 has K <= 2048)
  if constexpr (NB < 4) {
    if (steps <= 80) return launch_few_long<NB, 5, T>(p, st);
    return launch_few_long<NB, NB == 1 ? 9 : 6, T>(p, st);
  }
}

}  // namespace sd

using namespace sd;

extern "C" int specdec_linear_int8(const void* a, int64_t a_stride, const float* a_scale, const void* w,
                                   int64_t w_stride, const float* w_scale, const float* bias, void* out,
                                   int64_t out_stride, int32_t out_dtype, int64_t rows, int32_t width,
                                   int32_t out_features, int32_t weight_ready, int32_t* status,
                                   specdec_stream_t stream) {
  if (rows < 0 || rows > kMaxRows) return fail(SPECDEC_ERR_INVALID, "linear_int8: row count out of range");
  if (width <= 0 || width > kMaxWidth)
    return fail(SPECDEC_ERR_INVALID, "linear_int8: width must be in 1 .. %d", kMaxWidth);
  if (out_features <= 0 || out_features > (1 << 24))
    return fail(SPECDEC_ERR_INVALID, "linear_int8: out_features out of range");
  if (out_dtype != SPECDEC_F32 && out_dtype != SPECDEC_BF16)
    return fail(SPECDEC_ERR_INVALID, "linear_int8 writes float32 or bfloat16");
  if (rows == 0) return SPECDEC_OK;
  if (!a || !a_scale || !w || !w_scale || !out) return fail(SPECDEC_ERR_INVALID, "linear_int8: tensors must be CUDA");
  // the stride of a single row is of no account
  if (rows == 1) a_stride = (width + 15) & ~15, out_stride = out_features;
  if (out_features == 1) w_stride = (width + 15) & ~15;
  if (a_stride < width || w_stride < width || out_stride < out_features)
    return fail(SPECDEC_ERR_INVALID, "linear_int8: a row stride is smaller than its row");
  if ((a_stride | w_stride) & 15)
    return fail(SPECDEC_ERR_INVALID, "linear_int8: the row strides of the codes must be multiples of 16");
  if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(w)) & 15u)
    return fail(SPECDEC_ERR_INVALID, "linear_int8: the codes must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(w_scale) | reinterpret_cast<uintptr_t>(bias) |
       reinterpret_cast<uintptr_t>(status)) % 4 ||
      reinterpret_cast<uintptr_t>(out) % (out_dtype == SPECDEC_F32 ? 4 : 2))
    return fail(SPECDEC_ERR_INVALID, "linear_int8: a tensor is not aligned to its elements");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (few_rows(rows, width, out_features)) {
    const FewParams f = {static_cast<const int8_t*>(a), static_cast<const int8_t*>(w), a_scale, w_scale, bias, out,
                         a_stride, w_stride, out_stride, static_cast<int32_t>(rows), out_features, width, weight_ready};
    if (out_dtype == SPECDEC_F32)
      return rows <= 8 ? launch_few<1, float>(f, st) : rows <= 16 ? launch_few<2, float>(f, st) : launch_few<4, float>(f, st);
    return rows <= 8    ? launch_few<1, __nv_bfloat16>(f, st)
           : rows <= 16 ? launch_few<2, __nv_bfloat16>(f, st)
                        : launch_few<4, __nv_bfloat16>(f, st);
  }
  const int sms = device_sm_count();
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (int rc = allow_ring<1, __nv_bfloat16>(dev)) return rc;
  LinParams p = {};
  p.a_scale = a_scale;
  p.w_scale = w_scale;
  p.bias = bias;
  p.out = out;
  p.out_stride = out_stride;
  p.rows = static_cast<int32_t>(rows);
  p.n = out_features;
  p.chunks = (width + kLinChunk - 1) / kLinChunk;
  const LinShape shape = pick_shape(p.rows, p.n, p.chunks, sms, dev);
  p.tokens = shape.tokens;
  p.splits = shape.splits;
  p.ch_tiles = (p.n + shape.cg * kLinCh - 1) / (shape.cg * kLinCh);
  const int64_t units = static_cast<int64_t>(p.ch_tiles) * ((p.rows + p.tokens - 1) / p.tokens);
  if (units > (1 << 30)) return fail(SPECDEC_ERR_INVALID, "linear_int8: too many outputs");
  p.units = static_cast<int32_t>(units);
  p.weight_ready = weight_ready;
  p.status = status;
  p.wait_ns = wait_limit_ns();
  const int esize = out_dtype == SPECDEC_F32 ? 4 : 2;
  p.vec_out = (reinterpret_cast<uintptr_t>(out) % (4 * esize)) == 0 && out_stride % 4 == 0;
  p.rows16 = (reinterpret_cast<uintptr_t>(out) | static_cast<uintptr_t>(out_stride * esize) | static_cast<uintptr_t>(out_features) * esize) % 16 == 0;
  const int stage = kLinWTile + p.tokens / shape.cg * kLinChunk;
  const int pushed = p.splits > 1 ? p.tokens * kLinCh * 4 : 0;
  const int most = (kLinRing - pushed) / stage;
  p.stages = most < kLinMaxStages ? most : kLinMaxStages;
  p.tmem_cols = 32;
  while (p.tmem_cols < 2 * p.tokens) p.tmem_cols *= 2;
  CUtensorMap amap, wmap;
  if (int rc = encode_codes(&amap, a, width, rows, a_stride, p.tokens / shape.cg)) return rc;
  if (int rc = encode_codes(&wmap, w, width, out_features, w_stride, kLinCh)) return rc;
  const int smem = p.stages * stage + pushed + 1024;
  if (shape.cg == 2) {
    const int grid = 2 * (p.units < sms / 2 ? p.units : sms / 2);
    return out_dtype == SPECDEC_F32 ? launch_linear<2, float>(p, amap, wmap, grid, smem, dev, st)
                                    : launch_linear<2, __nv_bfloat16>(p, amap, wmap, grid, smem, dev, st);
  }
  const int grid = p.splits > 1 ? p.units * p.splits : (p.units < sms ? p.units : sms);
  return out_dtype == SPECDEC_F32 ? launch_linear<1, float>(p, amap, wmap, grid, smem, dev, st)
                                  : launch_linear<1, __nv_bfloat16>(p, amap, wmap, grid, smem, dev, st);
}
