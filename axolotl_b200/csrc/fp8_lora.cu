// A projection in 8-bit blocks with an adapter (ops/fp8.py) as one host call each way: a short training row spends less time on the device
// than the interpreter needs to issue the launches one by one (960 x 4096 by 6144, rank 16, forward and backward: kernels 106 us; 253 us
// with them issued from Python, 175 like this, 49 of it autograd's own).
#include "axb_common.cuh"

extern "C" int axb_gemm_skinny(const void* P, long long ldp, const void* S, long long lds, void* C, long long ldc, int R, int N,
                               int K, const void* P2, long long ldp2, const void* S2, long long lds2, int K2, float alpha,
                               const void* bias, int out_mode, int out_f32, int glu_kind, float glu_limit, int p_dep, int splits,
                               int pdl, int* status, void* stream);
extern "C" int axb_lora_bwd_dy(const void* dy, long long ld_dy, const void* B, long long ld_b, const void* xa, long long ld_xa, float* t32,
                               float* dB32, long long ldb32, int T, int N, int R, const int* blocks, int n_lora_blocks, int* status,
                               void* stream);
extern "C" int axb_fp8_low_pays(int T, int K);
extern "C" int axb_fp8_quantize_low(const void* x, long long ldx, const void* A, long long lda, void* q, long long ldq, float* s, long long lds,
                                    void* xa, long long ldxa, int T, int K, int R, float scale, int* status, void* stream);
extern "C" int axb_fp8_linear(const void* x, long long ldx, void* q, const void* W, long long ldw, const float* sw, long long sw_n,
                              long long sw_k, int b_mn, void* y, int T, int N, int K, const void* X2, long long ldx2, const void* B2,
                              long long ldb2, int K2, int tile, int* status, void* stream);
extern "C" int axb_fp8_adapter_grad(const void* q, long long ldq, const float* s, long long lds, const void* g, long long ldg, void* out,
                                    long long ldo, int T, int K, int R, int kind, int* status, void* stream);

namespace {

// bf16 of `scale` times a and of b, one after the other in memory (n4 and m4 groups of four): t and the gradient of B in one launch
__global__ void __launch_bounds__(256) fp8_lora_cast_kernel(const float4* __restrict__ a, const float4* __restrict__ b, uint2* __restrict__ a16,
                                                            uint2* __restrict__ b16, long long n4, long long m4, float scale) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n4 + m4) return;
  const float4 v = i < n4 ? a[i] : b[i - n4];
  const float s = i < n4 ? scale : 1.f;
  const uint2 o = make_uint2(pack_bf16x2(v.x * s, v.y * s), pack_bf16x2(v.z * s, v.w * s));
  if (i < n4) a16[i] = o;
  else b16[i - n4] = o;
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
  void* xa;                // scaling x A^T, bf16 [T, R]: written by the forward pass, read by the backward pass
  void* y;                 // y [T, N], or dx [T, K] (null: not wanted)
  const void* qx;          // backward: 8-bit rows of x
  float* t32;              // backward scratch: [T, R] fp32, [T, R] bf16
  void* t;
  void* dA;                // [R, K] (null: not wanted), fp32 or, where dA_bf16 is set, bf16
  float* dB;               // fp32 [N, R]; both are added to where add_* is set, else written
  void* dB16;              // its bf16 copy (null: none; dB is then scratch without gaps)
  const int* blocks;       // diagonal blocks of B
  int* status;
  long long ldx, ldw, sw_n, sw_k, lda, ldb, ldda, lddb;
  int T, N, K, R, tile, n_blocks, add_dA, add_dB, dA_bf16;
  float scaling;
};
static_assert(sizeof(AxbFp8Lora) == 16 * 8 + 8 * 8 + 10 * 4, "no gaps");

extern "C" int axb_fp8_lora_fwd(const AxbFp8Lora* l, void* stream) {
  if (l->T <= 0) return 0;
  const bool one = l->q && l->R <= 64 && axb_fp8_low_pays(l->T, l->K);         // xa and the 8-bit rows in one pass over x
  int rc;
  if (one) {
    const long long ldq = (l->K + 15ll) & ~15ll;
    rc = axb_fp8_quantize_low(l->x, l->ldx, l->A, l->lda, l->q, ldq, reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(l->q) + ldq * l->T),
                              (l->T + 3ll) & ~3ll, l->xa, l->R, l->T, l->K, l->R, l->scaling, l->status, stream);
  } else {
    rc = axb_gemm_skinny(l->x, l->ldx, l->A, l->lda, l->xa, l->R, l->T, l->R, l->K, nullptr, 0, nullptr, 0, 0, l->scaling, nullptr, 1, 0, 0,
                         0.f, 1, 0, 0, l->status, stream);
  }
  return rc ? rc : axb_fp8_linear(one ? nullptr : l->x, l->ldx, l->q, l->W, l->ldw, l->sw, l->sw_n, l->sw_k, 0, l->y, l->T, l->N, l->K, l->xa,
                                  l->R, l->B, l->ldb, l->R, l->tile, l->status, stream);
}

extern "C" int axb_fp8_lora_bwd(const AxbFp8Lora* l, void* stream) {
  if (l->T <= 0) return 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const long long n = (long long)l->T * l->R;
  const bool joined = !l->add_dB && l->dB == l->t32 + n && l->lddb == l->R;     // one block of zeros
  cudaError_t e = cudaMemsetAsync(l->t32, 0, (n + (joined ? (long long)l->N * l->R : 0)) * sizeof(float), st);
  if (e == cudaSuccess && !joined && !l->add_dB) e = cudaMemset2DAsync(l->dB, l->lddb * sizeof(float), 0, l->R * sizeof(float), l->N, st);
  if (e != cudaSuccess) return (int)e;
  int rc = axb_lora_bwd_dy(l->x, l->ldx, l->B, l->ldb, l->xa, l->R, l->t32, l->dB, l->lddb, l->T, l->N, l->R, l->blocks, l->n_blocks,
                           l->status, stream);
  if (rc) return rc;
  const long long n4 = n / 4, m4 = l->dB16 ? (long long)l->N * l->R / 4 : 0;      // R is a multiple of 8
  fp8_lora_cast_kernel<<<(unsigned)((n4 + m4 + 255) / 256), 256, 0, st>>>((const float4*)l->t32, (const float4*)l->dB, (uint2*)l->t,
                                                                           (uint2*)l->dB16, n4, m4, l->scaling);
  rc = (int)cudaGetLastError();
  if (!rc && l->y)
    rc = axb_fp8_linear(l->x, l->ldx, l->q, l->W, l->ldw, l->sw, l->sw_k, l->sw_n, 1, l->y, l->T, l->K, l->N, l->t, l->R, l->A, l->lda, l->R,
                        l->tile, l->status, stream);
  if (!rc && l->dA) {
    const long long ldq = (l->K + 15ll) & ~15ll, lds = (l->T + 3ll) & ~3ll;      // the layout of axb_fp8_linear
    rc = axb_fp8_adapter_grad(l->qx, ldq, reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(l->qx) + ldq * l->T), lds, l->t,
                              l->R, l->dA, l->ldda, l->T, l->K, l->R, l->dA_bf16 ? 2 : l->add_dA, l->status, stream);
  }
  return rc;
}
