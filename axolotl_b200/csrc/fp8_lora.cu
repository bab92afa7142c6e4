// A projection in 8-bit blocks with an adapter (ops/fp8.py) as one host call each way: a short training row spends less time on the device
// than the interpreter needs to issue the launches one by one (960 x 4096 by 6144, rank 16, forward and backward: kernels 104 us, 98 replayed
// from a graph; 253 us with them issued from Python, 166 like this, 49 of it autograd's own). Both ways, rank 48 in three blocks, fp32 masters,
// gradients into flat buffers: 152 us (106 replayed), 8192 rows 494; rank 32 by 28672 313 and 2119.
#include "axb_common.cuh"

extern "C" int axb_gemm_skinny(const void* P, long long ldp, const void* S, long long lds, void* C, long long ldc, int R, int N,
                               int K, const void* P2, long long ldp2, const void* S2, long long lds2, int K2, float alpha,
                               const void* bias, int out_mode, int out_f32, int glu_kind, float glu_limit, int p_dep, int splits,
                               int pdl, int* status, void* stream);
extern "C" int axb_lora_bwd_dy_parts(const void* dy, long long ld_dy, const void* B, long long ld_b, const void* xa, const void* xa_lo,
                                     long long ld_xa, float* t_parts, float* dB_parts, int T, int N, int R, const int* blocks,
                                     int n_lora_blocks, int splits, int* status, void* stream);
extern "C" int axb_fp8_low_pays(int T, int K, int R);
extern "C" int axb_fp8_quantize_low(const void* x, long long ldx, const void* A, long long lda, void* q, long long ldq, float* s, long long lds,
                                    void* xa, void* xa_lo, long long ldxa, int T, int K, int R, float scale, int* status, void* stream);
extern "C" int axb_fp8_linear(const void* x, long long ldx, void* q, const void* W, long long ldw, const float* sw, long long sw_n,
                              long long sw_k, int b_mn, void* y, int T, int N, int K, const void* X2, long long ldx2, const void* B2,
                              long long ldb2, int K2, int tile, int* status, void* stream);
extern "C" int axb_fp8_adapter_grad(const void* q, long long ldq, const float* s, long long lds, const void* g, const void* g_lo,
                                    long long ldg, void* out, long long ldo, int T, int K, int R, int kind, int* status, void* stream);

namespace {

constexpr int JOIN_ROWS = 8192;           // rows of dy whose parts are there at once (16 row chunks of csrc/lora_fused.cu)

struct JoinParams {
  const float4* t_parts;                  // [splits][T, R]
  const float4* dB_parts;                 // [chunks][N, R]; nothing outside the diagonal blocks
  uint2* t;                               // scale x the sum [T, R] as two bf16 numbers
  uint2* t_lo;
  const float* dB_old;                    // what the sum is added to (null: nothing); row strides ld
  float* dB;                              // fp32 (null: none)
  uint2* dB16;                            // bf16 [N, R] (null: none)
  long long ld;
  int T, N, R, splits, chunks, n_blocks;
  int row0[8], rows[8], r0[8], r[8];
  float scale;
};

// The sum of `count` parts at p, p + stride, .. by four lanes (l, l + 8, l + 16, l + 24), each every fourth of them, then across the lanes:
// the same order every time.
AXB_DEVICE float4 join4(const float4* p, long long stride, int count, bool any) {
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (any) {
#pragma unroll 4
    for (int s = (threadIdx.x & 31) >> 3; s < count; s += 4) {
      const float4 v = __ldg(p + s * stride);
      a.x += v.x;
      a.y += v.y;
      a.z += v.z;
      a.w += v.w;
    }
  }
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) {
    a.x += __shfl_xor_sync(0xffffffffu, a.x, o);
    a.y += __shfl_xor_sync(0xffffffffu, a.y, o);
    a.z += __shfl_xor_sync(0xffffffffu, a.z, o);
    a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
  }
  return a;
}

// t and the gradient of B from the parts of csrc/lora_fused.cu, four neighbouring values of a row for four lanes. Bound: the parts' bytes,
// most of them still in the L2 (dy 8192 x 4096, rank 16: 9 x 0.5 MB of t, 16 x 0.3 MB of B, 5 us; 8192 x 6144, rank 48: 20 MB, 11 us).
__global__ void __launch_bounds__(256) fp8_lora_join_kernel(const __grid_constant__ JoinParams p) {
  const int lane = threadIdx.x & 31, q = p.R >> 2;
  const long long n = (long long)p.T * q, n8 = (n + 7) & ~7ll, m = (long long)p.N * q;
  const long long u = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * 8 + (lane & 7);      // a warp is all t or all B
  if (u < n8) {
    const float4 a = join4(p.t_parts + u, n, p.splits, u < n);
    if (lane < 8 && u < n) {
      uint2 h, l;
      h.x = split_bf16x2(a.x * p.scale, a.y * p.scale, l.x);
      h.y = split_bf16x2(a.z * p.scale, a.w * p.scale, l.y);
      p.t[u] = h;
      p.t_lo[u] = l;
    }
    return;
  }
  const long long i = u - n8;
  const int row = (int)(i / q), c = (int)(i % q) * 4;
  int lo = 0, hi = 0;                     // columns of this row's block
  for (int b = 0; b < p.n_blocks; ++b)
    if (i < m && row >= p.row0[b] && row < p.row0[b] + p.rows[b]) {
      lo = p.r0[b];
      hi = p.r0[b] + p.r[b];
    }
  const bool any = c < hi && c + 4 > lo;
  const float4 a = join4(p.dB_parts + i, m, p.chunks, any);
  if (lane >= 8 || i >= m) return;
  const float in[4] = {a.x, a.y, a.z, a.w};
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    v[j] = (c + j >= lo && c + j < hi ? in[j] : 0.f) + (p.dB_old ? p.dB_old[row * p.ld + c + j] : 0.f);
  if (p.dB) {
    float* o = p.dB + row * p.ld + c;
    if ((p.ld & 3) == 0 && (reinterpret_cast<uintptr_t>(p.dB) & 15) == 0) {
      *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = v[j];
    }
  }
  if (p.dB16) p.dB16[i] = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

}  // namespace

// Packed by ops/fp8.py in this order.
struct AxbFp8Lora {
  const void* x;           // forward: x [T, K]; backward: dy [T, N]; bf16, row stride ldx
  void* q;                 // its 8-bit rows (axb_fp8_linear; null in a forward pass that keeps none)
  const void* W;           // codes [N, K], rows of ldw bytes, and their scales sw[n / 128][k / 128]
  const float* sw;
  const void* A;           // bf16 [R, K], [N, R]
  const void* B;
  void* xa;                // scaling x A^T, bf16 [T, R]: written by the forward pass, read by the backward pass. two: what that leaves of the
                           // fp32 sums, in bf16, T rows behind it
  void* y;                 // y [T, N], or dx [T, K] (null: not wanted)
  const void* qx;          // backward: 8-bit rows of x
  float* t_parts;          // backward scratch: fp32 [splits][min(T, 8192), R], [ceil of that many rows / 512][N, R]; bf16 [2][T, R]
  float* dB_parts;
  void* t;
  void* dA;                // [R, K] (null: not wanted), fp32 or, where dA_bf16 is set, bf16
  float* dB;               // fp32 [N, R]; both are added to where add_* is set, else written
  void* dB16;              // bf16 [N, R] instead of dB (null: none; dB is then scratch of row stride R, wanted beyond 8192 rows)
  const int* blocks;       // diagonal blocks of B
  int* status;
  long long ldx, ldw, sw_n, sw_k, lda, ldb, ldda, lddb;
  int T, N, K, R, tile, n_blocks, splits, add_dA, add_dB, dA_bf16;
  float scaling;
  int two;                 // always in a backward pass
};
static_assert(sizeof(AxbFp8Lora) == 17 * 8 + 8 * 8 + 12 * 4, "no gaps");

extern "C" int axb_fp8_lora_fwd(const AxbFp8Lora* l, void* stream) {
  if (l->T <= 0) return 0;
  const bool one = l->q && l->R <= 64 && axb_fp8_low_pays(l->T, l->K, l->R);   // xa and the 8-bit rows in one pass over x
  int rc;
  if (one) {
    const long long ldq = (l->K + 15ll) & ~15ll;
    rc = axb_fp8_quantize_low(l->x, l->ldx, l->A, l->lda, l->q, ldq, reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(l->q) + ldq * l->T),
                              (l->T + 3ll) & ~3ll, l->xa, l->two ? static_cast<char*>(l->xa) + 2ll * l->T * l->R : nullptr,
                              l->R, l->T, l->K, l->R, l->scaling, l->status, stream);
  } else {
    rc = axb_gemm_skinny(l->x, l->ldx, l->A, l->lda, l->xa, l->R, l->T, l->R, l->K, nullptr, 0, nullptr, 0, 0, l->scaling, nullptr, 1,
                         l->two ? 2 : 0, 0, 0.f, 1, 0, 0, l->status, stream);
  }
  return rc ? rc : axb_fp8_linear(one ? nullptr : l->x, l->ldx, l->q, l->W, l->ldw, l->sw, l->sw_n, l->sw_k, 0, l->y, l->T, l->N, l->K, l->xa,
                                  l->R, l->B, l->ldb, l->R, l->tile, l->status, stream);
}

extern "C" int axb_fp8_lora_bwd(const AxbFp8Lora* l, void* stream) {
  if (l->T <= 0) return 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (l->n_blocks < 1 || l->n_blocks > 8 || (l->T > JOIN_ROWS && !l->dB)) return -2;
  int rc = 0;
  const long long n = (long long)l->T * l->R;
  JoinParams p = {};
  p.t_parts = reinterpret_cast<const float4*>(l->t_parts);
  p.dB_parts = reinterpret_cast<const float4*>(l->dB_parts);
  p.ld = l->dB16 ? l->R : l->lddb;
  p.N = l->N;
  p.R = l->R;
  p.splits = l->splits;
  p.n_blocks = l->n_blocks;
  p.scale = l->scaling;
  for (int b = 0; b < l->n_blocks; ++b) {
    p.row0[b] = l->blocks[4 * b];
    p.rows[b] = l->blocks[4 * b + 1];
    p.r0[b] = l->blocks[4 * b + 2];
    p.r[b] = l->blocks[4 * b + 3];
  }
  for (int row = 0; row < l->T && !rc; row += JOIN_ROWS) {        // the parts of 8192 rows at a time: some 64 N R bytes of scratch
    const bool first = row == 0, last = l->T - row <= JOIN_ROWS;
    p.T = last ? l->T - row : JOIN_ROWS;
    p.chunks = (p.T + 511) / 512;
    const long long at = (long long)row * l->R;
    rc = axb_lora_bwd_dy_parts(static_cast<const char*>(l->x) + 2ll * row * l->ldx, l->ldx, l->B, l->ldb,
                               static_cast<const char*>(l->xa) + 2 * at, static_cast<const char*>(l->xa) + 2 * (n + at), l->R, l->t_parts,
                               l->dB_parts, p.T, l->N, l->R, l->blocks, l->n_blocks, l->splits, l->status, stream);
    if (rc) break;
    p.t = reinterpret_cast<uint2*>(static_cast<char*>(l->t) + 2 * at);
    p.t_lo = reinterpret_cast<uint2*>(static_cast<char*>(l->t) + 2 * (n + at));
    p.dB_old = first && (l->dB16 || !l->add_dB) ? nullptr : l->dB;
    p.dB = l->dB16 && last ? nullptr : l->dB;
    p.dB16 = last ? reinterpret_cast<uint2*>(l->dB16) : nullptr;
    const long long groups = (((long long)p.T * (p.R >> 2) + 7) & ~7ll) + (long long)p.N * (p.R >> 2);
    fp8_lora_join_kernel<<<(unsigned)((groups + 63) / 64), 256, 0, st>>>(p);
    rc = (int)cudaGetLastError();
  }
  if (!rc && l->y)
    rc = axb_fp8_linear(l->x, l->ldx, l->q, l->W, l->ldw, l->sw, l->sw_k, l->sw_n, 1, l->y, l->T, l->K, l->N, l->t, l->R, l->A, l->lda, l->R,
                        l->tile, l->status, stream);
  if (!rc && l->dA) {
    const long long ldq = (l->K + 15ll) & ~15ll, lds = (l->T + 3ll) & ~3ll;      // the layout of axb_fp8_linear
    rc = axb_fp8_adapter_grad(l->qx, ldq, reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(l->qx) + ldq * l->T), lds, l->t,
                              static_cast<const char*>(l->t) + 2 * n, l->R, l->dA, l->ldda, l->T, l->K, l->R,
                              l->dA_bf16 ? 2 : l->add_dA, l->status, stream);
  }
  return rc;
}
