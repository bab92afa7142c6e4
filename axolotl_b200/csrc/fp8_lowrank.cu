// The 8-bit rows of x [T, K] (csrc/fp8_rows.cu) and, in the same pass, xa = s x A^T [T, R] of the values as they came: what a projection in
// 8-bit blocks with an adapter needs of its input, which is then read once.
//
// Bound: HBM, 2 bytes read and 1 written per value. A step is 128 rows x 128 columns: bulk copies bring it in as the K-major 128-row
// operand of tcgen05.mma (A's block is the other one, N = 16 .. 64), and eight warps read the same tile back for the codes, a
// conflict-free 16 bytes a lane. They hand the stage back as soon as the values are in registers. K is split over a cluster, whose partial
// products meet in distributed shared memory in a fixed order. What it measures: 8192 x 14336, rank 16, 67 us: 5.9 TB/s and some 7 us of
// start, join and end (rank 48, with a stage less, 73); 960 x 4096 12.3 us. No faster: eight quantising warps of eight passes, five stages for
// one CTA of an SM.
#include "fp8_rows.cuh"

namespace {

constexpr int FL_WARPS = 16;              // that quantise
constexpr int FL_ROWS = 128 / FL_WARPS;   // rows of each
static_assert(FL_ROWS == 8, "four passes of two rows");
constexpr int FL_T = 64 + 32 * FL_WARPS;  // TMA, MMA, quantising warps
constexpr int FL_X = 128 * 256;           // x of a step: two chunks of 64 columns

struct Fp8LowParams {
  uint8_t* q;
  float* s;
  __nv_bfloat16* xa;
  __nv_bfloat16* xa_lo;                   // what the bf16 xa leaves, in bf16 (null: not wanted)
  long long ldq, lds, ldxa;
  int T, K, R;
  float scale;
  int* status;
};

template <int NR>
struct FlCfg {
  static constexpr int STAGE = FL_X + NR * 256;
  static constexpr int STAGES = NR <= 16 ? 3 : 2;         // two CTAs of an SM
  static constexpr int SMEM = STAGES * STAGE + 1024 + 128;
  static_assert(NR * 128 * 4 <= STAGE, "the partial product reuses the ring");
};

template <int NR>
__global__ void __launch_bounds__(FL_T, 2)
    fp8_quantize_low_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA, const Fp8LowParams p) {
  using C = FlCfg<NR>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE);
  uint64_t* empty = full + C::STAGES;     // the product's and the quantising warps'
  uint64_t* done = empty + C::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
  const int rank = (int)cluster_ctarank(), cs = (int)cluster_nctarank();
  const long long row0 = (long long)(blockIdx.x / cs) * 128;
  const int nk = (p.K + 127) / 128;
  const int kb0 = (int)((long long)nk * rank / cs), kb1 = (int)((long long)nk * (rank + 1) / cs);

  if (tid == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1 + FL_WARPS);
    }
    mbar_init(done, 1);
    mbar_fence_init();
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmA);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, NR < 32 ? 32 : NR);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();                // the product of these rows may set itself up meanwhile

  if (warp == 0) {
    int s = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!warp_all(mbar_wait(&empty[s], phase ^ 1, p.status, AXB_TIMEOUT_EMPTY))) break;
      if (elect_one()) {
        uint8_t* dst = smem + s * C::STAGE;
        mbar_expect_tx(&full[s], C::STAGE);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          tma_load_2d(dst + h * (FL_X / 2), &tmX, &full[s], kb * 128 + h * 64, (int)row0);
          tma_load_2d(dst + FL_X + h * (NR * 128), &tmA, &full[s], kb * 128 + h * 64, 0);
        }
      }
      __syncwarp();
      if (++s == C::STAGES) {
        s = 0;
        phase ^= 1;
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = make_idesc_bf16(128, NR, 0, 0);
    const uint64_t base = make_smem_desc_sw128(smem_u32(smem), 16, 1024);
    int s = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!warp_all(mbar_wait(&full[s], phase, p.status, AXB_TIMEOUT_FULL))) break;
      tc_fence_after();
      const uint64_t x = base + (uint32_t)(s * (C::STAGE / 16)), a = x + FL_X / 16;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)    // 16 columns each
          umma_f16(tmem, x + (kk >> 2) * (FL_X / 2 / 16) + (kk & 3) * 2, a + (kk >> 2) * (NR * 128 / 16) + (kk & 3) * 2, idesc,
                   kb > kb0 || kk > 0 ? 1u : 0u);
        umma_commit(&empty[s]);
        if (kb == kb1 - 1) umma_commit(done);
      }
      __syncwarp();
      if (++s == C::STAGES) {
        s = 0;
        phase ^= 1;
      }
    }
  } else {
    // sixteen lanes hold the block of a row, two rows a pass; this warp's rows start at r0
    const int r0 = (warp - 2) * FL_ROWS, half = lane >> 4, sub = lane & 15;
    int s = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!warp_all(mbar_wait(&full[s], phase, p.status, AXB_TIMEOUT_FULL))) break;
      const uint8_t* src = smem + s * C::STAGE + (sub >> 3) * (FL_X / 2);
      Eight<__nv_bfloat16> v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = r0 + 2 * i + half;
        v[i].raw[0] = *reinterpret_cast<const uint4*>(src + r * 128 + (((sub & 7) ^ (r & 7)) << 4));
      }
      uint2 w[4];
      int e[4];
      codes4(v, w, e);
      const int c = kb * 128 + sub * 8;
      uint32_t mine = 0;                  // lane l < 8: the exponent of row r0 + l
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long row = row0 + r0 + 2 * i + half;
        // rows of codes are padded to 16 bytes, so a vector that begins inside a row ends inside its padding
        if (row < p.T && c < p.K) *reinterpret_cast<uint2*>(p.q + row * p.ldq + c) = w[i];
        const uint32_t both = __shfl_sync(0xffffffffu, (uint32_t)e[i], (lane & 1) * 16);
        if (lane >> 1 == i) mine = both;
      }
      // The stage is handed back by a lane that a vote on the exponents names, so the arrival cannot pass the loads. (With lane 0 and a
      // __syncwarp behind the loads some of them saw the next contents of the stage.)
      if (lane == (__any_sync(0xffffffffu, mine > 255u) ? 1 : 0)) mbar_arrive(&empty[s]);
      if (lane < FL_ROWS && row0 + r0 + lane < p.T) p.s[(long long)kb * p.lds + row0 + r0 + lane] = __uint_as_float(mine << 23);
      if (++s == C::STAGES) {
        s = 0;
        phase ^= 1;
      }
    }
  }
  __syncwarp();
  warp_all(mbar_wait(done, 0, p.status, AXB_TIMEOUT_TMEM_FULL));
  tc_fence_after();
  __syncthreads();                        // every warp has left the ring
  float* part = reinterpret_cast<float*>(smem);          // partial product, [column][128 rows]
  if (warp >= 2 && warp < 6) {
#pragma unroll
    for (int c = 0; c < NR / 16; ++c) {
      uint32_t v[16];
      tmem_ld_32x16(tmem + (uint32_t((warp & 3) * 32) << 16) + c * 16, v);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) part[(c * 16 + j) * 128 + (warp & 3) * 32 + lane] = __uint_as_float(v[j]);
    }
  }
  tc_fence_before();
  if (cs > 1) cluster_sync();
  else __syncthreads();
  const uint32_t pbase = smem_u32(part);
  for (int i = rank * FL_T + tid; i < p.R * 16; i += cs * FL_T) {          // a row and eight columns
    const int r = i & 127, c = (i >> 7) * 8;
    if (row0 + r >= p.T) continue;
    float a[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = 0.f;
    for (int k = 0; k < cs; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] += cs == 1 ? part[(c + j) * 128 + r] : ld_cluster_f32(mapa_u32(pbase + ((c + j) * 128 + r) * 4, k));
    uint32_t o[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = split_bf16x2(a[2 * j] * p.scale, a[2 * j + 1] * p.scale, l[j]);
    *reinterpret_cast<uint4*>(p.xa + (row0 + r) * p.ldxa + c) = make_uint4(o[0], o[1], o[2], o[3]);
    if (p.xa_lo) *reinterpret_cast<uint4*>(p.xa_lo + (row0 + r) * p.ldxa + c) = make_uint4(l[0], l[1], l[2], l[3]);
  }
  if (cs > 1) cluster_sync();             // peers may still read this CTA's partial product
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, NR < 32 ? 32 : NR);
  }
}

template <int NR>
int launch_fp8_quantize_low(const CUtensorMap& x, const CUtensorMap& a, const Fp8LowParams& p, int tiles, int splits, cudaStream_t st) {
  auto kern = fp8_quantize_low_kernel<NR>;
  static std::atomic<unsigned long long> allowed{0};
  if (const int rc = axb_allow_smem((const void*)kern, FlCfg<NR>::SMEM, allowed)) return rc;
  AxbLaunch l(dim3((unsigned)(tiles * splits)), FL_T, FlCfg<NR>::SMEM, st, splits, false);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, x, a, p);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

// CTAs of a tile: eight while every cluster gets SMs to itself (14 of them), four elsewhere; two blocks at least to each CTA
int fp8_low_splits(int tiles, int nk) { return tiles <= 14 && nk >= 16 ? 8 : nk >= 8 ? 4 : nk >= 4 ? 2 : 1; }

}  // namespace

// Whether one pass beats the quantiser and a low-rank product of its own (both over x). One pass: 1.09 us for each block of a CTA and each
// CTA that an SM holds (148 SMs take 35 clusters of four), and 9.1 us around them, whatever the rank. Two: 10.6 us, 0.79 for a million values
// and 0.087 for each column of xa. By least squares over 300 shapes of 16 to 8192 rows, 2048 to 14336 columns and ranks 8 to 64 (x not in the
// L2); what it picks is 0.2 % above the better one on average, 10 % at most. Microseconds, one / two, rank 16: 64 x 14336 22.7 / 14.5,
// 960 x 4096 14.4 / 14.4, 960 x 14336 24.6 / 22.5, 2000 x 14336 39.0 / 33.3, 5000 x 4096 24.7 / 26.3, 8192 x 14336 67.8 / 102.6; rank 48:
// 700 x 8192 18.6 / 21.3, 2000 x 4096 18.5 / 22.5, 2000 x 14336 41.1 / 38.3, 8192 x 4096 28.9 / 43.0.
extern "C" int axb_fp8_low_pays(int T, int K, int R) {
  const int tiles = (T + 127) / 128, nk = (K + 127) / 128, splits = fp8_low_splits(tiles, nk);
  const double load = splits == 8 || tiles <= 35 ? 1. : tiles <= 70 ? 2. : tiles / 35.;
  return 9.1 + 1.09 * load * ((nk + splits - 1) / splits) <= 10.6 + 0.79e-6 * T * K + 0.087 * R;
}

// x: bf16 [T, K], row stride ldx; A: bf16 [R, K], row stride lda, R <= 64 and a multiple of 8; q: codes, rows of ldq bytes; s: fp32 [ceil(K /
// 128)][lds]; xa: bf16 [T, R], row stride ldxa; xa_lo: the same, what xa leaves of the fp32 sums (null: not wanted). x, A, q, xa and xa_lo start
// on 16 bytes and have row strides of whole 16 bytes.
extern "C" int axb_fp8_quantize_low(const void* x, long long ldx, const void* A, long long lda, void* q, long long ldq, float* s, long long lds,
                                    void* xa, void* xa_lo, long long ldxa, int T, int K, int R, float scale, int* status, void* stream) {
  if (T <= 0 || K <= 0) return 0;
  auto bad = [](const void* a, long long bytes) { return (reinterpret_cast<uintptr_t>(a) & 15) != 0 || (bytes & 15) != 0; };
  if (R <= 0 || R > 64 || (R & 7) || bad(x, 2 * ldx) || bad(A, 2 * lda) || bad(q, ldq) || bad(xa, 2 * ldxa) || bad(xa_lo, 0)
      || ldq < K || lds < T)
    return -2;
  const int NR = R <= 16 ? 16 : (R <= 32 ? 32 : 64);
  CUtensorMap tX, tA;
  int rc = axb_make_tmap_2d(&tX, x, T, K, ldx, 128, 64);
  if (!rc) rc = axb_make_tmap_2d(&tA, A, R, K, lda, NR, 64);
  if (rc) return -100 - rc;
  Fp8LowParams p = {};
  p.q = reinterpret_cast<uint8_t*>(q);
  p.s = s;
  p.xa = reinterpret_cast<__nv_bfloat16*>(xa);
  p.xa_lo = reinterpret_cast<__nv_bfloat16*>(xa_lo);
  p.ldq = ldq;
  p.lds = lds;
  p.ldxa = ldxa;
  p.T = T;
  p.K = K;
  p.R = R;
  p.scale = scale;
  p.status = status;
  const int tiles = (T + 127) / 128, splits = fp8_low_splits(tiles, (K + 127) / 128);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (NR == 16) return launch_fp8_quantize_low<16>(tX, tA, p, tiles, splits, st);
  if (NR == 32) return launch_fp8_quantize_low<32>(tX, tA, p, tiles, splits, st);
  return launch_fp8_quantize_low<64>(tX, tA, p, tiles, splits, st);
}
