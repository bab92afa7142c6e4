// dA[r, k] (+)= sum_t g[t, r] x8[t, k]: the gradient of an adapter's A from the 8-bit rows that the forward pass kept (codes q [T, K] and
// scales s[k / 128][t], csrc/fp8_rows.cu) and g [T, R] = s dy B in bf16.
//
// Bound: one pass over the codes (HBM), half of what the bf16 rows would take. The scales lie along the contracted axis, so the codes
// are widened first: eight warps turn a tile of 64 rows x 128 columns into bf16 (exact: four significant bits and a power of two) as the
// MN-major 128-row operand of tcgen05.mma, g is the other one, 64 of its columns at a time; TWO: g comes as two bf16 numbers, and both
// products go to the same sums. The rows are split over a cluster whose partial
// sums meet in distributed shared memory in a fixed order: no atomics, the same bits every time.
// What it measures: 8192 x 14336, rank 16, 57 us (2 TB/s of codes; expanding the rows and a bf16 product took 122), bound by the integer
// pipe of the SMs that hold two of the 224 CTAs, some seven instructions a code; 8192 x 11008 41.5 us, 8192 x 4096 20.6. With g as two numbers
// and a stage less 66 us, 8192 x 4096, rank 48, 25.
#include "axb_common.cuh"

namespace {

constexpr int FA_T = 320;                 // TMA, MMA, eight widening warps
constexpr int FA_ROWS = 64;               // rows of a step
constexpr int FA_Q = FA_ROWS * 128;       // codes of a step
constexpr int FA_G = FA_ROWS * 128;       // g of a step: 64 columns in bf16
constexpr int FA_X = FA_ROWS * 256;       // widened tile: two chunks of 64 columns
constexpr int FA_XBUFS = 2;
constexpr int FA_S = FA_ROWS * 4;         // scales of a step
template <bool TWO>
struct FaCfg {
  static constexpr int STAGES = TWO ? 3 : 4;            // two CTAs of an SM
  static constexpr int STAGE = FA_Q + FA_G * (TWO ? 2 : 1);
  static constexpr int SMEM = STAGES * (STAGE + FA_S) + FA_XBUFS * FA_X + 1024 + 256;
  static_assert(64 * 128 * 4 <= STAGES * STAGE, "the partial tile reuses the ring");
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two CTAs of an SM");
};

struct Fp8AdapterParams {
  float* out;
  __nv_bfloat16* out16;     // instead of out: the sums rounded once
  long long ldo;
  int T, K, R, accumulate, vec;
  int* status;
};

// Two E4M3 codes, each in the upper byte of a half word, as bf16 values times `sc`: sign, exponent and mantissa are moved to their bf16
// places, which reads the number with an exponent 120 too low, and both multiplications are exact. Conversion instructions (e4m3 -> f16 ->
// f32 -> bf16) run at a fraction of the rate and bound the kernel: 8192 x 14336 rows, rank 16, 58 us with them.
AXB_DEVICE uint32_t widen2(uint32_t h, __nv_bfloat162 sc) {
  const uint32_t bits = ((h & 0x7F007F00u) >> 4) | (h & 0x80008000u);
  const uint32_t up = 0x7B807B80u;          // 2^120, twice
  __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&bits), *reinterpret_cast<const __nv_bfloat162*>(&up));
  v = __hmul2(v, sc);
  return *reinterpret_cast<uint32_t*>(&v);
}

template <int NR, bool TWO>
__global__ void __launch_bounds__(FA_T, 2)
    fp8_adapter_grad_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmS,
                            const __grid_constant__ CUtensorMap tmG, const __grid_constant__ CUtensorMap tmL, const Fp8AdapterParams p) {
  constexpr int FA_STAGES = FaCfg<TWO>::STAGES, FA_STAGE = FaCfg<TWO>::STAGE;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sX = smem + FA_STAGES * FA_STAGE;
  float* sS = reinterpret_cast<float*>(sX + FA_XBUFS * FA_X);
  uint64_t* full = reinterpret_cast<uint64_t*>(sS + FA_STAGES * FA_ROWS);   // codes, scales and g have arrived
  uint64_t* empty = full + FA_STAGES;                                   // the product that read g has ended
  uint64_t* xfull = empty + FA_STAGES;                                  // widened by eight warps
  uint64_t* xempty = xfull + FA_XBUFS;
  uint64_t* done = xempty + FA_XBUFS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
  const int rank = (int)cluster_ctarank(), cs = (int)cluster_nctarank();
  const int tile = blockIdx.x / cs, r0 = blockIdx.y * 64;
  const int steps = (p.T + FA_ROWS - 1) / FA_ROWS;
  const int t0 = (int)((long long)steps * rank / cs), t1 = (int)((long long)steps * (rank + 1) / cs);

  if (tid == 0) {
    for (int s = 0; s < FA_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < FA_XBUFS; ++s) {
      mbar_init(&xfull[s], 8);
      mbar_init(&xempty[s], 1);
    }
    mbar_init(done, 1);
    mbar_fence_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmG);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, NR < 32 ? 32 : NR);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    int s = 0;
    uint32_t phase = 0;
    for (int t = t0; t < t1; ++t) {
      if (!warp_all(mbar_wait(&empty[s], phase ^ 1, p.status, AXB_TIMEOUT_EMPTY))) break;
      if (elect_one()) {
        uint8_t* dst = smem + s * FA_STAGE;
        mbar_expect_tx(&full[s], FA_STAGE + FA_S);
        tma_load_2d(sS + s * FA_ROWS, &tmS, &full[s], t * FA_ROWS, tile);
        tma_load_2d(dst, &tmQ, &full[s], tile * 128, t * FA_ROWS);
        tma_load_2d(dst + FA_Q, &tmG, &full[s], r0, t * FA_ROWS);
        if constexpr (TWO) tma_load_2d(dst + FA_Q + FA_G, &tmL, &full[s], r0, t * FA_ROWS);
      }
      __syncwarp();
      if (++s == FA_STAGES) {
        s = 0;
        phase ^= 1;
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = make_idesc_bf16(128, NR, 1, 1);
    const uint64_t base_x = make_smem_desc_sw128(smem_u32(sX), FA_X / 2, 1024);
    const uint64_t base_g = make_smem_desc_sw128(smem_u32(smem + FA_Q), 16, 1024);
    int s = 0, b = 0;
    uint32_t phase = 0;
    for (int t = t0; t < t1; ++t) {
      // the widening warps have waited for the stage's copies; this warp's own wait makes g visible to its product
      if (!warp_all(mbar_wait(&xfull[b], phase, p.status, AXB_TIMEOUT_GENERIC) &&
                    mbar_wait(&full[s], (uint32_t)((t - t0) / FA_STAGES) & 1, p.status, AXB_TIMEOUT_FULL)))
        break;
      tc_fence_after();
      const uint64_t x = base_x + (uint32_t)(b * (FA_X / 16)), g = base_g + (uint32_t)(s * (FA_STAGE / 16));
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < FA_ROWS / 16; ++kk)
          umma_f16(tmem, x + kk * (2048 / 16), g + kk * (2048 / 16), idesc, t > t0 || kk > 0 ? 1u : 0u);
        if constexpr (TWO) {
#pragma unroll
          for (int kk = 0; kk < FA_ROWS / 16; ++kk) umma_f16(tmem, x + kk * (2048 / 16), g + (FA_G + kk * 2048) / 16, idesc, 1u);
        }
        umma_commit(&empty[s]);
        umma_commit(&xempty[b]);
        if (t == t1 - 1) umma_commit(done);
      }
      __syncwarp();
      if (++s == FA_STAGES) s = 0;
      if (++b == FA_XBUFS) {
        b = 0;
        phase ^= 1;
      }
    }
  } else {
    // 16 codes of a row at a time: this thread's rows are r and 32 + r of a step
    const int w = tid - 64, r = w >> 3, c16 = w & 7;
    int s = 0, b = 0;
    uint32_t phase = 0, xphase = 0;
    for (int t = t0; t < t1; ++t) {
      if (!warp_all(mbar_wait(&full[s], phase, p.status, AXB_TIMEOUT_FULL) &&
                    mbar_wait(&xempty[b], xphase ^ 1, p.status, AXB_TIMEOUT_EMPTY)))
        break;
      const uint8_t* src = smem + s * FA_STAGE;
      uint8_t* dst = sX + b * FA_X + (c16 >> 2) * (FA_X / 2);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = i * 32 + r;
        const uint4 q = *reinterpret_cast<const uint4*>(src + row * 128 + c16 * 16);
        const uint32_t in[4] = {q.x, q.y, q.z, q.w};
        uint32_t o[8], nan = 0;
        const __nv_bfloat162 sc = __float2bfloat162_rn(sS[s * FA_ROWS + row]);   // a power of two (0 behind the last row)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          nan |= (in[j] & 0x7F7F7F7Fu) + 0x01010101u;
          o[2 * j] = widen2(__byte_perm(in[j], 0u, 0x1404), sc);
          o[2 * j + 1] = widen2(__byte_perm(in[j], 0u, 0x3424), sc);
        }
        if (nan & 0x80808080u) {                   // a code 0x7F or 0xFF among the sixteen
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (((in[j >> 1] >> (16 * (j & 1) + 8 * h)) & 0x7Fu) == 0x7Fu) o[j] |= 0x7FFFu << (16 * h);
        }
        uint8_t* to = dst + row * 128;
        const int j0 = (c16 & 3) * 2;
        *reinterpret_cast<uint4*>(to + ((j0 ^ (row & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(to + (((j0 + 1) ^ (row & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&xfull[b]);
      if (++s == FA_STAGES) {
        s = 0;
        phase ^= 1;
      }
      if (++b == FA_XBUFS) {
        b = 0;
        xphase ^= 1;
      }
    }
  }
  __syncwarp();
  warp_all(mbar_wait(done, 0, p.status, AXB_TIMEOUT_TMEM_FULL));
  tc_fence_after();
  __syncthreads();                        // every warp has left the ring
  float* part = reinterpret_cast<float*>(smem);          // partial tile, [r][128 columns]
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
  const int rows = min(p.R - r0, 64);
  for (int i = rank * FA_T + tid; i < rows * 32; i += cs * FA_T) {
    const int rr = i >> 5, c = (i & 31) * 4, k = tile * 128 + c;
    if (k >= p.K) continue;
    float4 u[8], a = make_float4(0.f, 0.f, 0.f, 0.f);    // all on their way before the first is added
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q < cs) u[q] = cs == 1 ? *reinterpret_cast<const float4*>(part + rr * 128 + c) : ld_cluster_f32x4(mapa_u32(pbase + (rr * 128 + c) * 4, q));
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q < cs) {
        a.x += u[q].x;
        a.y += u[q].y;
        a.z += u[q].z;
        a.w += u[q].w;
      }
    if (p.out16) {
      __nv_bfloat16* o = p.out16 + (long long)(r0 + rr) * p.ldo + k;
      if (p.vec && k + 4 <= p.K) {
        *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
      } else {
        const float v[4] = {a.x, a.y, a.z, a.w};
        for (int j = 0; j < 4 && k + j < p.K; ++j) o[j] = __float2bfloat16(v[j]);
      }
      continue;
    }
    float* o = p.out + (long long)(r0 + rr) * p.ldo + k;
    if (p.vec && k + 4 <= p.K) {
      if (p.accumulate) {
        const float4 b = *reinterpret_cast<const float4*>(o);
        a.x += b.x;
        a.y += b.y;
        a.z += b.z;
        a.w += b.w;
      }
      *reinterpret_cast<float4*>(o) = a;
    } else {
      const float v[4] = {a.x, a.y, a.z, a.w};
      for (int j = 0; j < 4 && k + j < p.K; ++j) o[j] = v[j] + (p.accumulate ? o[j] : 0.f);
    }
  }
  if (cs > 1) cluster_sync();             // peers may still read this CTA's partial tile
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, NR < 32 ? 32 : NR);
  }
}

template <int NR, bool TWO>
int launch_adapter_grad(const CUtensorMap& q, const CUtensorMap& sc, const CUtensorMap& g, const CUtensorMap& lo, const Fp8AdapterParams& p,
                        int tiles, int chunks, int splits, cudaStream_t st) {
  auto kern = fp8_adapter_grad_kernel<NR, TWO>;
  static std::atomic<unsigned long long> allowed{0};
  if (const int rc = axb_allow_smem((const void*)kern, FaCfg<TWO>::SMEM, allowed)) return rc;
  AxbLaunch l(dim3((unsigned)(tiles * splits), (unsigned)chunks), FA_T, FaCfg<TWO>::SMEM, st, splits, false);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, q, sc, g, lo, p);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace

// q: codes [T, K], rows of ldq bytes; s: fp32 [ceil(K / 128)][lds]; g: bf16 [T, R], row stride ldg; g_lo: the same, added to it (null: none);
// out: [R, K], row stride ldo; kind 0: fp32, written, 1: fp32, added to, 2: bf16, written. q, s, g and g_lo start on 16 bytes and have row
// strides of whole 16 bytes.
extern "C" int axb_fp8_adapter_grad(const void* q, long long ldq, const float* s, long long lds, const void* g, const void* g_lo,
                                    long long ldg, void* out, long long ldo, int T, int K, int R, int kind, int* status, void* stream) {
  if (K <= 0 || R <= 0) return 0;
  auto bad = [](const void* v, long long bytes) { return (reinterpret_cast<uintptr_t>(v) & 15) != 0 || (bytes & 15) != 0; };
  if (T <= 0 || bad(q, ldq) || bad(s, 4 * lds) || bad(g, 2 * ldg) || bad(g_lo, 0) || lds < T || ldo < K) return -2;
  CUtensorMap tQ, tS, tG, tL;
  int rc = axb_make_tmap_2d(&tQ, q, T, K, ldq, FA_ROWS, 128, 1, false);
  if (!rc) rc = axb_make_tmap_2d(&tS, s, (K + 127) / 128, T, lds, 1, FA_ROWS, 4, false);
  if (!rc) rc = axb_make_tmap_2d(&tG, g, T, R, ldg, FA_ROWS, 64);
  tL = tG;
  if (!rc && g_lo) rc = axb_make_tmap_2d(&tL, g_lo, T, R, ldg, FA_ROWS, 64);
  if (rc) return -100 - rc;
  const int tiles = (K + 127) / 128, chunks = (R + 63) / 64, steps = (T + FA_ROWS - 1) / FA_ROWS;
  if (chunks > 65535) return -2;
  const int splits = axb_cluster_split((long long)tiles * chunks, steps);
  Fp8AdapterParams p = {};
  p.out = reinterpret_cast<float*>(out);
  p.out16 = kind == 2 ? reinterpret_cast<__nv_bfloat16*>(out) : nullptr;
  p.ldo = ldo;
  p.T = T;
  p.K = K;
  p.R = R;
  p.accumulate = kind == 1;
  p.vec = (ldo & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  p.status = status;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto run = [&](auto one, auto two) { return (g_lo ? two : one)(tQ, tS, tG, tL, p, tiles, chunks, splits, st); };
  if (R <= 16) return run(launch_adapter_grad<16, false>, launch_adapter_grad<16, true>);
  if (R <= 32) return run(launch_adapter_grad<32, false>, launch_adapter_grad<32, true>);
  return run(launch_adapter_grad<64, false>, launch_adapter_grad<64, true>);
}
