// y[t, n] = sum_b sx[t, b] sw[n / 128, b] (sum_{k in b} q[t, k] w[n, k]) (+ sum_r a2[t, r] b2[n, r]) for at most 64 tokens: a generation
// step through a frozen weight in 8-bit blocks (codes [N, K], csrc/fp8_gemm.cu).
//
// Bound: one pass over the codes (HBM). The weight is the 128-row operand of tcgen05.mma (kind::f8f6f4), so no tensor-core row is
// padding, and the tokens are its N = 16 .. 64 columns. The K range of a tile is split over a cluster of up to 8 CTAs and two CTAs share
// an SM, so that some 160 KB of codes per SM are in flight; the partial tiles meet in distributed shared memory in a fixed order.
// Every block of 128 columns starts an accumulator of its own; four warps (a thread owns a weight row) add it to sums in registers,
// times the weight's scale and the token's. The rows come as codes (csrc/fp8_rows.cu), or (FUSED) in bf16: then four warps quantise them
// into the operand tile while the weight's bulk copies arrive, and the codes and their scales never reach memory. ops/fp8.py says when.
// On quantised rows it is a dependent launch of the kernel that quantised them. One token by 4096 x 4096 8.3 us (codes in the L2), by
// 4096 x 28672 25 us (4.7 TB/s); 64 tokens, 14336 x 4096, 20 us.
#include <cuda_fp8.h>

#include "axb_common.cuh"

namespace {

constexpr int FS_T = 320;                 // TMA, MMA, four summing warps, four quantising warps
constexpr int FS_P = 128 * 128;           // weight tile of a block
constexpr int FS_RING = 16;               // blocks whose row scales are held (stages + accumulators + 1 at most are in use)

struct Fp8SkinnyParams {
  const __nv_bfloat16* x;
  const __nv_bfloat16* x2;                // bf16 extension of the tokens
  const float* sx;                        // scales of quantised rows [block][ldsx] (FUSED: not there)
  const float* sw;
  __nv_bfloat16* y;
  long long ldx, ldx2, ldsx, sw_n, sw_k, ldy;
  int T, N, K, K2, vec;                   // vec: rows of x start on 16 bytes
  int* status;
};

template <int NT>
struct FsCfg {
  static constexpr int STAGE = FS_P + NT * 128;
  static constexpr int STAGES = NT <= 32 ? 5 : 4;
  static constexpr int BUFS = 4;
  static constexpr int SCALES = FS_RING * NT * 4;
  static constexpr int BYTES = STAGES * STAGE;
  static constexpr int SMEM = BYTES + SCALES + 1024 + 512;
  static_assert(NT * 128 * 4 <= BYTES, "the partial tile reuses the ring");
  static_assert(STAGES + BUFS + 1 <= FS_RING, "row scales outlive their block");
};

AXB_DEVICE uint4 ldg16(const __nv_bfloat16* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

// 16 values of a row from column c on (zero past K)
AXB_DEVICE void load16(const Fp8SkinnyParams& p, const __nv_bfloat16* row, int c, uint32_t (&v)[8]) {
  if (p.vec && c + 16 <= p.K) {
    const uint4 a = ldg16(row + c), b = ldg16(row + c + 8);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t lo = c + 2 * j < p.K ? (uint32_t)__bfloat16_as_ushort(row[c + 2 * j]) : 0u;
      const uint32_t hi = c + 2 * j + 1 < p.K ? (uint32_t)__bfloat16_as_ushort(row[c + 2 * j + 1]) : 0u;
      v[j] = lo | (hi << 16);
    }
  }
}

template <int NT, bool FUSED>
__global__ void __launch_bounds__(FS_T, 2)
    fp8_skinny_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmB2, const __grid_constant__ CUtensorMap tmX,
                      const __grid_constant__ CUtensorMap tmX2, const Fp8SkinnyParams p) {
  using C = FsCfg<NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* scales = reinterpret_cast<float*>(smem + C::BYTES);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BYTES + C::SCALES);   // the copy's and the quantising warps'
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint64_t* tempty = tfull + C::BUFS;
  uint64_t* ready = tempty + C::BUFS;                                          // row scales of a block are in the ring
  uint64_t* freed = ready + FS_RING;                                           // and have been used (where the rows come quantised)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(freed + FS_RING);
  const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
  const int rank = (int)cluster_ctarank(), cs = (int)cluster_nctarank();
  const int tile = blockIdx.x / cs;
  const int nk_main = (p.K + 127) / 128, nk = nk_main + (p.K2 + 63) / 64;
  const int kb0 = (int)((long long)nk * rank / cs), kb1 = (int)((long long)nk * (rank + 1) / cs);

  if (tid == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], FUSED ? 5 : 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < C::BUFS; ++s) {
      mbar_init(&tfull[s], 1);
      mbar_init(&tempty[s], 4);
    }
    for (int s = 0; s < FS_RING; ++s) {
      mbar_init(&ready[s], 4);
      mbar_init(&freed[s], 4);
    }
    mbar_fence_init();
    tma_prefetch_desc(&tmW);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::BUFS * NT);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  float* part = reinterpret_cast<float*>(smem);     // partial tile, [token][128], in the ring after the last product

  if (warp == 0) {
    auto load_w = [&](int kb, int s) {
      const bool ext = kb >= nk_main;
      mbar_expect_tx(&full[s], FUSED ? FS_P : C::STAGE);
      tma_load_2d(smem + s * C::STAGE, ext ? &tmB2 : &tmW, &full[s], ext ? (kb - nk_main) * 64 : kb * 128, tile * 128);
    };
    auto load_x = [&](int kb, int s) {
      const bool ext = kb >= nk_main;
      if (!FUSED) tma_load_2d(smem + s * C::STAGE + FS_P, ext ? &tmX2 : &tmX, &full[s], ext ? (kb - nk_main) * 64 : kb * 128, 0);
    };
    // the weight does not come from the launch before this one: its first tiles are requested while the rows are quantised
    const int pre = min(C::STAGES, kb1 - kb0);
    for (int i = 0; i < pre; ++i) {
      if (elect_one()) load_w(kb0 + i, i);
      __syncwarp();
    }
    pdl_wait();
    for (int i = 0; i < pre; ++i) {
      if (elect_one()) load_x(kb0 + i, i);
      __syncwarp();
    }
    int s = 0;
    uint32_t phase = 0;                   // stage s is refilled once its first contents have been used
    for (int kb = kb0 + pre; kb < kb1; ++kb) {
      if (!warp_all(mbar_wait(&empty[s], phase, p.status, AXB_TIMEOUT_EMPTY))) break;
      if (elect_one()) {
        load_w(kb, s);
        load_x(kb, s);
      }
      __syncwarp();
      if (++s == C::STAGES) {
        s = 0;
        phase ^= 1;
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t id8 = (1u << 4) | (uint32_t(NT >> 3) << 17) | (uint32_t(128 >> 4) << 24);   // E4M3 (format 0), fp32 accumulator
    constexpr uint32_t id16 = make_idesc_bf16(128, NT, 0, 0);
    const uint64_t base = make_smem_desc_sw128(smem_u32(smem), 16, 1024);
    int s = 0, buf = 0;
    uint32_t phase = 0, buf_phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!warp_all(mbar_wait(&full[s], phase, p.status, AXB_TIMEOUT_FULL) &&
                    mbar_wait(&tempty[buf], buf_phase ^ 1, p.status, AXB_TIMEOUT_TMEM_EMPTY)))
        break;
      tc_fence_after();
      const uint64_t a = base + (uint32_t)(s * (C::STAGE / 16)), b = a + FS_P / 16;
      const uint32_t d = tmem + buf * NT;
      if (elect_one()) {
        if (kb < nk_main) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) umma_f8(d, a + kk * 2, b + kk * 2, id8, kk > 0 ? 1u : 0u);
        } else {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) umma_f16(d, a + kk * 2, b + kk * 2, id16, kk > 0 ? 1u : 0u);
        }
        umma_commit(&empty[s]);
        umma_commit(&tfull[buf]);
      }
      __syncwarp();
      if (++s == C::STAGES) {
        s = 0;
        phase ^= 1;
      }
      if (++buf == C::BUFS) {
        buf = 0;
        buf_phase ^= 1;
      }
    }
  } else if (warp < 6) {
    const float* sw = p.sw + (long long)tile * p.sw_n;
    const uint32_t t_base = tmem + (uint32_t((warp & 3) * 32) << 16);
    uint64_t sum[NT / 2];                 // two tokens each
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) sum[j] = 0ull;
    float mine = 0.f;                     // lane l: the weight's scale of block kb0 + l, kb0 + 32 + l, ..
    int buf = 0;
    uint32_t buf_phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0;
      if ((i & 31) == 0) mine = kb + lane < nk_main ? __ldg(sw + (kb + lane) * p.sw_k) : 1.f;
      const float w = __shfl_sync(0xffffffffu, mine, i & 31);
      const uint64_t ww = pack_f32x2(w, w);
      if (!warp_all(mbar_wait(&tfull[buf], buf_phase, p.status, AXB_TIMEOUT_TMEM_FULL) &&
                    mbar_wait(&ready[i % FS_RING], (uint32_t)(i / FS_RING) & 1, p.status, AXB_TIMEOUT_GENERIC)))
        break;
      tc_fence_after();
      const float4* sx = reinterpret_cast<const float4*>(scales + (i % FS_RING) * NT);
#pragma unroll
      for (int c = 0; c < NT / 16; ++c) {
        uint32_t r[16];
        tmem_ld_32x16(t_base + buf * NT + c * 16, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 s4 = sx[c * 4 + j];
          uint64_t* to = sum + c * 8 + 2 * j;
          to[0] = fma_f32x2(pack_b32x2(r[4 * j], r[4 * j + 1]), mul_f32x2(ww, pack_f32x2(s4.x, s4.y)), to[0]);
          to[1] = fma_f32x2(pack_b32x2(r[4 * j + 2], r[4 * j + 3]), mul_f32x2(ww, pack_f32x2(s4.z, s4.w)), to[1]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&tempty[buf]);
        // a block late: this one's scales may still be on their way to the sums, which nothing orders before the arrival
        if (!FUSED && i > 0) mbar_arrive(&freed[(i - 1) % FS_RING]);
      }
      if (++buf == C::BUFS) {
        buf = 0;
        buf_phase ^= 1;
      }
    }
    // this warp has seen the last product end, and with it every read and write of the ring
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const float2 two = unpack_f32x2(sum[j >> 1]);
      if (j < p.T) part[j * 128 + (warp & 3) * 32 + lane] = j & 1 ? two.y : two.x;
    }
  } else if (!FUSED) {
    pdl_wait();
    // the rows' scales into the ring, a quarter of the tokens a warp, as far ahead as the ring goes. (Not by the operands' `empty`: nothing
    // keeps these warps within one phase of it.)
    const int t = (warp - 6) * (NT / 4) + lane;
    const bool mine = lane < NT / 4;
    auto fetch = [&](int kb) { return mine && kb < nk_main && t < p.T ? ld_after_wait(p.sx + kb * p.ldsx + t) : 1.f; };
    float next = fetch(kb0);
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0, slot = i % FS_RING;
      const float v = next;
      next = fetch(kb + 1);
      if (!warp_all(mbar_wait(&freed[slot], ((uint32_t)(i / FS_RING) & 1) ^ 1, p.status, AXB_TIMEOUT_EMPTY))) break;
      if (mine) scales[slot * NT + t] = v;
      __syncwarp();
      if (lane == 0) mbar_arrive(&ready[slot]);
    }
  } else {
    // eight lanes hold the block of a row (16 values each), four rows a pass; tokens past T leave their columns as they are
    const int sub = lane >> 3, at = lane & 7;
    constexpr int PASSES = NT / 16;
    uint32_t v[PASSES][8];
    auto fetch = [&](int kb) {
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int t = i * 16 + (warp - 6) * 4 + sub;
        if (t < p.T && kb < nk_main) load16(p, p.x + t * p.ldx, kb * 128 + at * 16, v[i]);
      }
    };
    fetch(kb0);
    int s = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0;
      if (!warp_all(mbar_wait(&empty[s], phase ^ 1, p.status, AXB_TIMEOUT_EMPTY))) break;
      uint8_t* tileS = smem + s * C::STAGE + FS_P;
      float* sx = scales + (i % FS_RING) * NT;
#pragma unroll
      for (int q = 0; q < PASSES; ++q) {
        const int t = q * 16 + (warp - 6) * 4 + sub;
        uint4 o;
        float scale = 1.f;
        if (kb < nk_main) {
          // the largest magnitude of a block, two values an instruction; NaN takes no part
          const bool live = t < p.T;
          __nv_bfloat162 m2 = __habs2(*reinterpret_cast<__nv_bfloat162*>(&v[q][0]));
#pragma unroll
          for (int j = 1; j < 8; ++j) m2 = __hmax2(m2, __habs2(*reinterpret_cast<__nv_bfloat162*>(&v[q][j])));
          float top = live ? __bfloat162float(__hmax(m2.x, m2.y)) : 0.f, f[16];
#pragma unroll
          for (int m = 4; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 u = unpack_bf16x2(v[q][j]);
            f[2 * j] = live ? u.x : 0.f;
            f[2 * j + 1] = live ? u.y : 0.f;
          }
          if (__any_sync(0xffffffffu, !(top <= 3.402823466e38f))) {
            top = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              if (fabsf(f[j]) <= 3.402823466e38f) top = fmaxf(top, fabsf(f[j]));
              else f[j] = __uint_as_float(0x7FC00000u);
            }
#pragma unroll
            for (int m = 4; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
          }
          const int e = fp8_scale_exponent(top);
          const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
          scale = __uint_as_float((uint32_t)e << 23);
          if (e >= 247) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (fabsf(f[j]) > 240.f * 0x1p120f) f[j] = copysignf(240.f * 0x1p120f, f[j]);
          }
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * j] * inv, f[4 * j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * j + 2] * inv, f[4 * j + 3] * inv), __NV_SATFINITE, __NV_E4M3);
            w[j] = lo | (hi << 16);
          }
          o = make_uint4(w[0], w[1], w[2], w[3]);
        } else {                          // eight bf16 of the extension
          const int c = (kb - nk_main) * 64 + at * 8;
          o = make_uint4(0u, 0u, 0u, 0u);
          if (t < p.T && c < p.K2) o = ldg16(p.x2 + t * p.ldx2 + c);
        }
        *reinterpret_cast<uint4*>(tileS + t * 128 + ((at ^ (t & 7)) << 4)) = o;
        if (at == 0) sx[t] = scale;
      }
      fetch(kb + 1);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&ready[i % FS_RING]);
        mbar_arrive(&full[s]);
      }
      if (++s == C::STAGES) {
        s = 0;
        phase ^= 1;
      }
    }
  }
  pdl_wait();                             // nothing is written before the launch before this one has ended
  if (cs > 1) cluster_sync();
  else __syncthreads();
  const uint32_t pbase = smem_u32(part);
  const bool vec = (p.ldy & 3) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 7) == 0;
  for (int i = rank * FS_T + tid; i < p.T * 32; i += cs * FS_T) {
    const int t = i >> 5, r = (i & 31) * 4, n = tile * 128 + r;
    if (n >= p.N) continue;
    float4 u[8], a = make_float4(0.f, 0.f, 0.f, 0.f);    // all on their way before the first is added
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q < cs) u[q] = cs == 1 ? *reinterpret_cast<const float4*>(part + t * 128 + r) : ld_cluster_f32x4(mapa_u32(pbase + (t * 128 + r) * 4, q));
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q < cs) {
        a.x += u[q].x;
        a.y += u[q].y;
        a.z += u[q].z;
        a.w += u[q].w;
      }
    __nv_bfloat16* y = p.y + (long long)t * p.ldy + n;
    if (vec && n + 4 <= p.N) {
      *reinterpret_cast<uint2*>(y) = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
    } else {
      const float o[4] = {a.x, a.y, a.z, a.w};
      for (int j = 0; j < 4 && n + j < p.N; ++j) y[j] = __float2bfloat16(o[j]);
    }
  }
  tc_fence_before();
  if (cs > 1) cluster_sync();             // peers may still read this CTA's partial tile
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::BUFS * NT);
  }
}

template <int NT, bool FUSED>
int launch_fp8_skinny(const CUtensorMap (&m)[4], const Fp8SkinnyParams& p, int tiles, int splits, cudaStream_t st) {
  auto kern = fp8_skinny_kernel<NT, FUSED>;
  static std::atomic<unsigned long long> allowed{0};
  if (const int rc = axb_allow_smem((const void*)kern, FsCfg<NT>::SMEM, allowed)) return rc;
  AxbLaunch l(dim3((unsigned)(tiles * splits)), FS_T, FsCfg<NT>::SMEM, st, splits, !FUSED);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, m[0], m[1], m[2], m[3], p);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace

// See the head of this file. x: bf16 [T, K], T <= 64; q (null: the rows are quantised by the kernel): their codes, rows of ldq bytes, and
// sx: their scales [ceil(K / 128)][ldsx]; W: codes [N, K], rows of ldw bytes, and their scales sw[(n / 128) * sw_n + b * sw_k]; y: bf16
// [T, N]; X2 [T, K2] and B2 [N, K2] bf16, K2 = 0: none. q, W, X2 and B2 start on 16 bytes and have row strides of whole 16 bytes.
extern "C" int axb_fp8_skinny(const void* x, long long ldx, const void* q, long long ldq, const float* sx, long long ldsx, const void* W,
                              long long ldw, const float* sw, long long sw_n, long long sw_k, void* y, long long ldy, int T, int N, int K,
                              const void* X2, long long ldx2, const void* B2, long long ldb2, int K2, int* status, void* stream) {
  if (T <= 0 || N <= 0) return 0;
  auto bad = [](const void* a, long long bytes) { return (reinterpret_cast<uintptr_t>(a) & 15) != 0 || (bytes & 15) != 0; };
  if (T > 64 || K <= 0 || bad(W, ldw) || (q && bad(q, ldq))) return -2;
  if (K2 > 0 && (bad(X2, 2 * ldx2) || bad(B2, 2 * ldb2) || (K2 & 7))) return -2;
  const int NT = T <= 16 ? 16 : (T <= 32 ? 32 : 64);
  CUtensorMap m[4];
  int rc = axb_make_tmap_2d(&m[0], W, N, K, ldw, 128, 128, 1);
  m[1] = m[2] = m[3] = m[0];
  if (!rc && K2 > 0) rc = axb_make_tmap_2d(&m[1], B2, N, K2, ldb2, 128, 64);
  if (!rc && q) rc = axb_make_tmap_2d(&m[2], q, T, K, ldq, NT, 128, 1);
  if (!rc && q && K2 > 0) rc = axb_make_tmap_2d(&m[3], X2, T, K2, ldx2, NT, 64);
  if (rc) return -100 - rc;
  Fp8SkinnyParams p = {};
  p.x = (const __nv_bfloat16*)x;
  p.x2 = (const __nv_bfloat16*)X2;
  p.sx = sx;
  p.sw = sw;
  p.y = (__nv_bfloat16*)y;
  p.ldx = ldx;
  p.ldx2 = ldx2;
  p.ldsx = ldsx;
  p.sw_n = sw_n;
  p.sw_k = sw_k;
  p.ldy = ldy;
  p.T = T;
  p.N = N;
  p.K = K;
  p.K2 = K2 > 0 ? K2 : 0;
  p.vec = !bad(x, 2 * ldx);
  p.status = status;
  const int tiles = (N + 127) / 128, nk = (K + 127) / 128 + (p.K2 + 63) / 64, splits = axb_cluster_split(tiles, nk);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (q) {
    if (NT == 16) return launch_fp8_skinny<16, false>(m, p, tiles, splits, st);
    if (NT == 32) return launch_fp8_skinny<32, false>(m, p, tiles, splits, st);
    return launch_fp8_skinny<64, false>(m, p, tiles, splits, st);
  }
  if (NT == 16) return launch_fp8_skinny<16, true>(m, p, tiles, splits, st);
  if (NT == 32) return launch_fp8_skinny<32, true>(m, p, tiles, splits, st);
  return launch_fp8_skinny<64, true>(m, p, tiles, splits, st);
}
