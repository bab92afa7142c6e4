// C[M, N] = A B^T (+ A2 B2^T) with A and B in E4M3 and scales for blocks of 128 along K:
//
//   C[m, n] = sum_b sA[b][m] sB[n / 128, b] (sum_{k in b} a[m, k] b[n, k]) + sum_r a2[m, r] b2[n, r]
//
// A: codes [M, K] with a scale per row and block (csrc/fp8_rows.cu); B: codes of a frozen weight with one fp32 scale per 128 x 128
// block, [N, K] (forward) or stored [K, N] (b_mn: the input gradient reads the same codes as an MN-major operand, no second copy).
// A2 / B2: bf16 K-extension, the low-rank update of an adapter, accumulated as further blocks of scale 1.
//
// The scales change every 128 columns of K, so an accumulator cannot stay in TMEM: the four MMAs of a block start a new one, and
// eight epilogue warps add it, times its scale, to fp32 sums in registers while the tensor cores work on the next. A thread owns a
// row: one scale for all its columns of a weight block.
// Tiles: 256 x 256 or 256 x 128 by a CTA pair, 128 x 128 by one CTA (ops/fp8.py says when). In the largest a block is two products of 128
// columns with two accumulators each (columns of both CTAs' B rows: 64 h .. of either), one for each half of the epilogue warps, so
// that one half drains its accumulator while the other's is computed; in the others one product with four.
//
// Bound: the epilogue's turn of a block. TMEM reads (110 cycles) and multiply-adds (250, half a packed one a cycle and partition) follow
// one another in a warp behind some 500 cycles of waits, arrivals and scale loads, against 512 of the tensor cores and as many of the
// operands' 64 bytes a cycle and SM. A 4096 x 8192 by 4096 product takes 205 k cycles; 147 k with the epilogue left out, 160 k with its
// reads or its arithmetic alone. 8192 x 4096 by 28672: 850 us, 2.26 PFLOP/s (940 to 1000 back to back under the power cap); the input gradient of
// 8192 x 14336 by 4096 440 us. No faster: 16 epilogue warps, scales through a ring of cp.async copies, two TMEM loads in flight, one
// product of 256 columns a block.
#include "axb_common.cuh"

extern "C" int axb_fp8_quantize_rows(const void* x, long long ldx, int dtype, void* q, long long ldq, float* s, long long lds,
                                     long long rows, int K, void* stream);
extern "C" int axb_fp8_skinny(const void* x, long long ldx, const void* q, long long ldq, const float* sx, long long ldsx, const void* W,
                              long long ldw, const float* sw, long long sw_n, long long sw_k, void* y, long long ldy, int T, int N, int K,
                              const void* X2, long long ldx2, const void* B2, long long ldb2, int K2, int* status, void* stream);

namespace {

constexpr int G_THREADS = 320;                 // TMA, MMA, eight epilogue warps
constexpr int G_BK = 128;                      // bytes of a K block: 128 codes, or 64 bf16 of the extension
constexpr int G_OP = 128 * G_BK;               // an operand tile of a CTA
constexpr int G_RING = 6 * 2 * G_OP;
constexpr int G_EPI = 8 * 4096;                // per epilogue warp: 32 rows x 64 bf16
constexpr int G_SMEM = G_RING + G_EPI + 1024 + 256;

struct Fp8GemmParams {
  const float* sa;
  const float* sb;
  long long ldsa, sb_n, sb_k;                  // scale of block b: sa[b * ldsa + m], sb[(n / 128) * sb_n + b * sb_k]
  __nv_bfloat16* C;
  long long ldc;
  int M, N, K, K2;
  int group_m, tma_store;
  int* status;
};

AXB_DEVICE void umma_f8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// MN-major tile in chunks of 64 codes: 64-byte rows, one k each, 64-byte swizzle (8-row atoms of 512 bytes); lbo = bytes between chunks.
AXB_DEVICE uint64_t make_smem_desc_sw64(uint32_t saddr, uint32_t lbo_bytes) {
  return (make_smem_desc_sw128(saddr, lbo_bytes, 512) & ~(7ull << 61)) | (4ull << 61);
}
// Instruction descriptor, kind::f8f6f4: E4M3 operands (format 0), fp32 accumulator.
AXB_DEVICE constexpr uint32_t make_idesc_e4m3(int m, int n, int b_mn_major) {
  return (1u << 4) | (uint32_t(b_mn_major) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

AXB_DEVICE const float* at_bytes(const float* p, long long n) { return reinterpret_cast<const float*>(reinterpret_cast<const char*>(p) + n); }

// tiles in bands of group_m tile rows that sweep over N together (their A rows stay in L2)
AXB_DEVICE void fp8_tile(int tile, int num_m, int num_n, int group_m, int& m_blk, int& n_blk) {
  const int per = group_m * num_n, group = tile / per, first = group * group_m;
  const int rows = min(num_m - first, group_m), in = tile - group * per;
  m_blk = first + in % rows;
  n_blk = in / rows;
}

template <int CTAS, int SETS, bool B_MN>
__global__ void __launch_bounds__(G_THREADS, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmA2, const __grid_constant__ CUtensorMap tmB2,
                    const __grid_constant__ CUtensorMap tmC, const Fp8GemmParams p) {
  constexpr bool PAIR = CTAS == 2;
  constexpr int TILE_M = 128 * CTAS, TILE_N = 128 * SETS;       // SETS products of 128 columns a block
  constexpr int BN = TILE_N / CTAS;            // columns whose B a CTA brings in
  constexpr int G_STAGE = G_OP + BN * G_BK, G_STAGES = G_RING / G_STAGE;
  constexpr int BUFS = 4 / SETS;               // accumulators of each product
  constexpr int GROUPS = SETS;                 // groups of 64 columns that an epilogue warp owns
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sEpi = smem + G_RING;
  uint64_t* full = reinterpret_cast<uint64_t*>(sEpi + G_EPI);   // leader's: both CTAs' loads of the stage
  uint64_t* empty = full + G_STAGES;                            // one per CTA
  uint64_t* tfull = empty + G_STAGES;                           // [set][buffer], one per CTA
  uint64_t* tempty = tfull + 4;                                 // leader's: the epilogue warps that read the accumulator
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 4);
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)cluster_ctarank() : 0;
  const int worker = blockIdx.x / CTAS, workers = gridDim.x / CTAS;
  const int num_m = (p.M + TILE_M - 1) / TILE_M, num_n = (p.N + TILE_N - 1) / TILE_N, tiles = num_m * num_n;
  const int nk_main = (p.K + 127) / 128, nk = nk_main + (p.K2 + 63) / 64;

  if (threadIdx.x == 0) {
    for (int s = 0; s < G_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&tfull[s], 1);
      mbar_init(&tempty[s], 8 * CTAS / SETS);
    }
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_slot, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();          // the barriers of both CTAs are ready before anything arrives on them
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();                                  // in a dependent launch: the rows have been quantised

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = worker; tile < tiles && ok; tile += workers) {
      int m_blk, n_blk;
      fp8_tile(tile, num_m, num_n, p.group_m, m_blk, n_blk);
      const int m0 = m_blk * TILE_M + rank * 128, n0 = n_blk * TILE_N + rank * BN;
      for (int kb = 0; kb < nk; ++kb) {
        if (!warp_all(mbar_wait(&empty[stage], phase ^ 1, p.status, AXB_TIMEOUT_EMPTY))) {
          ok = false;
          break;
        }
        const bool ext = kb >= nk_main;
        uint8_t* a = smem + stage * G_STAGE;
        uint8_t* b = a + G_OP;
        if (elect_one()) {
          auto load = [&](uint8_t* dst, const CUtensorMap* m, int c0, int c1) {
            if constexpr (PAIR) tma_load_2d_pair(dst, m, mapa_u32(smem_u32(&full[stage]), 0), c0, c1);
            else tma_load_2d(dst, m, &full[stage], c0, c1);
          };
          if (rank == 0) mbar_expect_tx(&full[stage], CTAS * G_STAGE);
          const CUtensorMap* mb = ext ? &tmB2 : &tmB;
          const int ka = ext ? (kb - nk_main) * 64 : kb * 128;
          load(a, ext ? &tmA2 : &tmA, ka, m0);
          if (B_MN) {
            load(b, mb, n0, ka);
            if (BN > 64) load(b + G_OP / 2, mb, n0 + 64, ka);
          } else {
            load(b, mb, ka, n0);
          }
        }
        __syncwarp();
        if (++stage == G_STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      constexpr uint32_t id8 = make_idesc_e4m3(TILE_M, 128, B_MN ? 1 : 0);
      constexpr uint32_t id16 = make_idesc_bf16(TILE_M, 128, 0, B_MN ? 1 : 0);
      const uint64_t base_a = make_smem_desc_sw128(smem_u32(smem), 16, 1024);
      // MN-major: two chunks of 64 columns (64-byte rows of codes, 128-byte rows of bf16), G_OP / 2 apart
      const uint64_t base_b8 = B_MN ? make_smem_desc_sw64(smem_u32(smem + G_OP), G_OP / 2) : base_a + G_OP / 16;
      const uint64_t base_b16 = B_MN ? make_smem_desc_sw128(smem_u32(smem + G_OP), G_OP / 2, 1024) : base_a + G_OP / 16;
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      bool ok = true;
      for (int tile = worker; tile < tiles && ok; tile += workers) {
        for (int kb = 0; kb < nk && ok; ++kb) {
          ok = warp_all(mbar_wait_spin(&full[stage], phase, p.status, AXB_TIMEOUT_FULL));
          if (!ok) break;
          const uint32_t at = (uint32_t)(stage * (G_STAGE / 16));
          const uint64_t a = base_a + at;
#pragma unroll
          for (int h = 0; h < SETS; ++h) {
            // the arrivals order no memory but the reads of TMEM: a release of every access in flight would wait for the scales that
            // were requested for the next block (4096 x 8192 by 4096: 257 us with it, 131 without)
            uint64_t* free = &tempty[h * BUFS + buf];
            ok = warp_all(PAIR ? mbar_wait_partner(free, buf_phase ^ 1, p.status, AXB_TIMEOUT_TMEM_EMPTY)
                               : mbar_wait_spin(free, buf_phase ^ 1, p.status, AXB_TIMEOUT_TMEM_EMPTY));
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tmem + (h * BUFS + buf) * 128;
            if (elect_one()) {
              if (kb < nk_main) {
                const uint64_t b = base_b8 + at + h * (G_OP / 2 / 16);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {  // 32 codes each
                  const uint64_t bk = b + kk * (B_MN ? 2048 / 16 : 2);
                  if constexpr (PAIR) umma_f8_pair(d, a + kk * 2, bk, id8, kk > 0 ? 1u : 0u);
                  else umma_f8(d, a + kk * 2, bk, id8, kk > 0 ? 1u : 0u);
                }
              } else {
                const uint64_t b = base_b16 + at + h * (G_OP / 2 / 16);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {  // 16 bf16 each
                  const uint64_t bk = b + kk * (B_MN ? 2048 / 16 : 2);
                  if constexpr (PAIR) umma_f16_pair(d, a + kk * 2, bk, id16, kk > 0 ? 1u : 0u);
                  else umma_f16(d, a + kk * 2, bk, id16, kk > 0 ? 1u : 0u);
                }
              }
              if constexpr (PAIR) {
                umma_commit_pair_mc(&tfull[h * BUFS + buf]);
                if (h == SETS - 1) umma_commit_pair_mc(&empty[stage]);
              } else {
                umma_commit(&tfull[h * BUFS + buf]);
                if (h == SETS - 1) umma_commit(&empty[stage]);
              }
            }
            __syncwarp();
          }
          if (++stage == G_STAGES) {
            stage = 0;
            phase ^= 1;
          }
          if (++buf == BUFS) {
            buf = 0;
            buf_phase ^= 1;
          }
        }
      }
    }
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    uint8_t* stg = sEpi + (warp - 2) * 4096;
    const int set = SETS == 2 ? half : 0;
    const uint32_t t_base = tmem + (uint32_t(quad * 32) << 16) + (SETS == 2 ? set * BUFS * 128 : half * 64);
    const long long step_a = p.ldsa * 4, step_b = p.sb_k * 4;   // bytes: the address arithmetic stays off the multipliers
    int buf = 0;
    uint32_t buf_phase = 0;
    bool ok = true;
    for (int tile = worker; tile < tiles && ok; tile += workers) {
      int m_blk, n_blk;
      fp8_tile(tile, num_m, num_n, p.group_m, m_blk, n_blk);
      const int row0 = m_blk * TILE_M + rank * 128 + quad * 32, row = row0 + lane;
      const int col0 = n_blk * TILE_N + half * 64;                // group g: col0 + 128 g ..
      const bool live = row < p.M;
      const float* sa = p.sa + (live ? row : 0);
      const float* sb = p.sb + (long long)(col0 >> 7) * p.sb_n;
      const float* sb2 = sb + (col0 + 128 < p.N ? p.sb_n : 0);  // of group 1
      uint64_t sum[GROUPS * 32];
#pragma unroll
      for (int j = 0; j < GROUPS * 32; ++j) sum[j] = 0ull;
      float na = ld_after_wait(sa), nb0 = __ldg(sb), nb1 = GROUPS > 1 ? __ldg(sb2) : 0.f;   // the next block's, requested a block ahead
      for (int kb = 0; kb < nk; ++kb) {
        const float s0 = na * nb0, s1 = na * nb1;
        na = nb0 = nb1 = 1.f;
        if (kb + 1 < nk_main) {
          sa = at_bytes(sa, step_a);
          sb = at_bytes(sb, step_b);
          na = ld_after_wait(sa);
          nb0 = __ldg(sb);
          if (GROUPS > 1) nb1 = __ldg(sb2 = at_bytes(sb2, step_b));
        }
        ok = warp_all(mbar_wait(&tfull[set * BUFS + buf], buf_phase, p.status, AXB_TIMEOUT_TMEM_FULL));
        if (!ok) break;
        tc_fence_after();
        // columns on their way at once: all 64 where the sums leave the registers for them (777 x 6144 by 4096 32.0 us, 32.8 with 16)
        constexpr int LD = GROUPS == 1 ? 64 : 16;
#pragma unroll
        for (int c = 0; c < GROUPS * 64; c += LD) {
          uint32_t r[LD];
#pragma unroll
          for (int l = 0; l < LD; l += 16) tmem_ld_32x16(t_base + buf * 128 + c + l, *reinterpret_cast<uint32_t(*)[16]>(r + l));
          tmem_ld_wait();
          if (c == GROUPS * 64 - LD) {         // the accumulator has been read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (PAIR) mbar_arrive_partner(mapa_u32(smem_u32(&tempty[set * BUFS + buf]), 0));
              else mbar_arrive(&tempty[buf]);
            }
          }
          const uint64_t sc = c < 64 ? pack_f32x2(s0, s0) : pack_f32x2(s1, s1);
#pragma unroll
          for (int j = 0; j < LD / 2; ++j) sum[c / 2 + j] = fma_f32x2(pack_b32x2(r[2 * j], r[2 * j + 1]), sc, sum[c / 2 + j]);
        }
        if (++buf == BUFS) {
          buf = 0;
          buf_phase ^= 1;
        }
      }
      if (!ok) break;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const int cc = col0 + g * 128;
        uint4 w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = unpack_f32x2(sum[g * 32 + j * 4 + e]);
            o[e] = pack_bf16x2(f.x, f.y);
          }
          w[j] = make_uint4(o[0], o[1], o[2], o[3]);
        }
        if (p.tma_store) {
          if (row0 < p.M && cc < p.N) {        // the same for the whole warp
            if (lane == 0) bulk_wait_group_read<0>();
            __syncwarp();
            stage_row128(stg, lane, w);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmC, stg, cc, row0);
              bulk_commit_group();
            }
          }
        } else if (live) {
          __nv_bfloat16* o = p.C + (long long)row * p.ldc + cc;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t q[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (cc + j * 8 + e < p.N) o[j * 8 + e] = __ushort_as_bfloat16((unsigned short)(q[e >> 1] >> (16 * (e & 1))));
          }
        }
      }
    }
    if (lane == 0) bulk_wait_group<0>();
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();          // neither CTA leaves while its partner still signals it
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

int fp8_sm_count() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 1 ? n : 148;
}

template <int CTAS, int SETS, bool B_MN>
int launch_fp8(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& a2, const CUtensorMap& b2, const CUtensorMap& c,
               const Fp8GemmParams& p, bool pdl, cudaStream_t st) {
  auto kern = fp8_gemm_kernel<CTAS, SETS, B_MN>;
  static std::atomic<unsigned long long> allowed{0};
  if (const int rc = axb_allow_smem((const void*)kern, G_SMEM, allowed)) return rc;
  const long long tiles = (long long)((p.M + 128 * CTAS - 1) / (128 * CTAS)) * ((p.N + 128 * SETS - 1) / (128 * SETS));
  const long long workers = tiles < fp8_sm_count() / CTAS ? tiles : fp8_sm_count() / CTAS;
  AxbLaunch l(dim3((unsigned)(workers * CTAS)), G_THREADS, G_SMEM, st, CTAS == 2 ? 2 : 0, pdl);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, a, b, a2, b2, c, p);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace

// See the head of this file. A: codes [M, K], rows of lda bytes; sa: fp32 [ceil(K / 128)][ldsa]; B: codes [N, K] (b_mn: [K, N]), rows of
// ldb bytes; sb: fp32, the scale of columns n and block b at sb[(n / 128) * sb_n + b * sb_k]; C: bf16 [M, N]; A2 [M, K2] and B2 [N, K2]
// (b_mn: [K2, N]) bf16, K2 = 0: none. Operands start on 16 bytes and have row strides of whole 16 bytes. pdl: the launch before this one
// is the one that quantised A; this one's start overlaps its end.
static int fp8_gemm_entry(const void* A, long long lda, const float* sa, long long ldsa, const void* B, long long ldb, const float* sb,
                          long long sb_n, long long sb_k, int b_mn, void* C, long long ldc, int M, int N, int K, const void* A2,
                            long long lda2, const void* B2, long long ldb2, int K2, int tile, bool pdl, int* status, void* stream) {
  if (M <= 0 || N <= 0) return 0;
  auto bad = [](const void* q, long long bytes) { return (reinterpret_cast<uintptr_t>(q) & 15) != 0 || (bytes & 15) != 0; };
  if (K <= 0 || bad(A, lda) || bad(B, ldb) || ldsa < M) return -2;
  if (K2 > 0 && (bad(A2, 2 * lda2) || bad(B2, 2 * ldb2))) return -2;
  const bool pair = tile != 128;
  const int bn = tile == 192 ? 64 : 128;
  CUtensorMap tA, tB, tA2, tB2, tC;
  int rc = axb_make_tmap_2d(&tA, A, M, K, lda, 128, 128, 1);
  if (!rc) rc = b_mn ? axb_make_tmap_2d(&tB, B, K, N, ldb, 128, 64, 1, false, true) : axb_make_tmap_2d(&tB, B, N, K, ldb, bn, 128, 1);
  tA2 = tC = tA;
  tB2 = tB;
  if (!rc && K2 > 0) {
    rc = axb_make_tmap_2d(&tA2, A2, M, K2, lda2, 128, 64);
    if (!rc) rc = b_mn ? axb_make_tmap_2d(&tB2, B2, K2, N, ldb2, 64, 64) : axb_make_tmap_2d(&tB2, B2, N, K2, ldb2, bn, 64);
  }
  const int tma_store = !bad(C, 2 * ldc);
  if (!rc && tma_store) rc = axb_make_tmap_2d(&tC, C, M, N, ldc, 32, 64);
  if (rc) return -100 - rc;
  Fp8GemmParams p = {};
  p.sa = sa;
  p.sb = sb;
  p.ldsa = ldsa;
  p.sb_n = sb_n;
  p.sb_k = sb_k;
  p.C = reinterpret_cast<__nv_bfloat16*>(C);
  p.ldc = ldc;
  p.M = M;
  p.N = N;
  p.K = K;
  p.K2 = K2 > 0 ? K2 : 0;
  p.tma_store = tma_store;
  p.status = status;
  const long long band = (20ll << 20) / ((pair ? 256ll : 128ll) * K);   // A rows of a band: about 20 MB of the L2
  p.group_m = (int)(band < 2 ? 2 : (band > 16 ? 16 : band));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto run = [&](auto kmajor, auto mnmajor) { return (b_mn ? mnmajor : kmajor)(tA, tB, tA2, tB2, tC, p, pdl, st); };
  if (tile == 256) return run(launch_fp8<2, 2, false>, launch_fp8<2, 2, true>);
  if (tile == 192) return run(launch_fp8<2, 1, false>, launch_fp8<2, 1, true>);
  return run(launch_fp8<1, 1, false>, launch_fp8<1, 1, true>);
}

extern "C" int axb_fp8_gemm(const void* A, long long lda, const float* sa, long long ldsa, const void* B, long long ldb, const float* sb,
                            long long sb_n, long long sb_k, int b_mn, void* C, long long ldc, int M, int N, int K, const void* A2,
                            long long lda2, const void* B2, long long ldb2, int K2, int tile, int* status, void* stream) {
  return fp8_gemm_entry(A, lda, sa, ldsa, B, ldb, sb, sb_n, sb_k, b_mn, C, ldc, M, N, K, A2, lda2, B2, ldb2, K2, tile, false, status, stream);
}

// y = x8 W8^T (b_mn: x8 W8) (+ X2 B2) of bf16 rows x [T, K] in one call. q: where the 8-bit rows go, T rows of K rounded up to 16 bytes and
// behind them the scales, fp32 [ceil(K / 128)][T rounded up to 4]; null: they are not kept (at most 64 rows, forward). x null: the launch
// before this one has put them there. The other arguments are those of axb_fp8_gemm.
extern "C" int axb_fp8_linear(const void* x, long long ldx, void* q, const void* W, long long ldw, const float* sw, long long sw_n,
                              long long sw_k, int b_mn, void* y, int T, int N, int K, const void* X2, long long ldx2, const void* B2,
                              long long ldb2, int K2, int tile, int* status, void* stream) {
  if (!q) {
    if (b_mn) return -2;
    return axb_fp8_skinny(x, ldx, nullptr, 0, nullptr, 0, W, ldw, sw, sw_n, sw_k, y, N, T, N, K, X2, ldx2, B2, ldb2, K2, status, stream);
  }
  const long long ldq = (K + 15ll) & ~15ll, lds = (T + 3ll) & ~3ll;
  float* s = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(q) + ldq * T);
  const int rc = x ? axb_fp8_quantize_rows(x, ldx, 0, q, ldq, s, lds, T, K, stream) : 0;
  if (rc) return rc;
  if (!b_mn && tile == 0)
    return axb_fp8_skinny(x, ldx, q, ldq, s, lds, W, ldw, sw, sw_n, sw_k, y, N, T, N, K, X2, ldx2, B2, ldb2, K2, status, stream);
  return fp8_gemm_entry(q, ldq, s, lds, W, ldw, sw, sw_n, sw_k, b_mn, y, N, T, N, K, X2, ldx2, B2, ldb2, K2, tile, true, status, stream);
}

// The arguments of axb_fp8_linear as ops/fp8.py packs them: a generation step's product takes the device 8 us and the host 12, of which
// the conversion of 21 arguments one by one was 2.7.
struct AxbFp8Linear {
  const void* x;
  void* q;
  const void* W;
  const float* sw;
  void* y;
  const void* X2;
  const void* B2;
  int* status;
  void* stream;
  long long ldx, ldw, sw_n, sw_k, ldx2, ldb2;
  int T, N, K, K2, tile, b_mn;
};
static_assert(sizeof(AxbFp8Linear) == 9 * 8 + 6 * 8 + 6 * 4, "no gaps");

extern "C" int axb_fp8_linear_packed(const AxbFp8Linear* a) {
  return axb_fp8_linear(a->x, a->ldx, a->q, a->W, a->ldw, a->sw, a->sw_n, a->sw_k, a->b_mn, a->y, a->T, a->N, a->K, a->X2, a->ldx2, a->B2,
                        a->ldb2, a->K2, a->tile, a->status, a->stream);
}
