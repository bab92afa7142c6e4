// Activations in 8 bits: E4M3 codes with one power-of-two scale for each row and 128 columns.
//
//   s[b][t] = 2^ceil(log2(max |x[t, 128 b ..]| / 448))   (1 for a block of zeros, never below 2^-126),   q = rn_e4m3(x / s)
//
// A power of two makes x / s exact, so that a code is the nearest E4M3 number whatever the precision it is computed in, and q s exact
// in bf16 (four significant bits): what comes back is what every product of the codes has seen. NaN and infinities become NaN codes
// and take no part in the maximum, so their neighbours keep their values. A finite value stays finite: where the nearest code would
// stand for 2^128 it is the one below.
// Scales are stored [block][row]: a GEMM's thread owns a row of the accumulator and reads its scale beside its neighbours'.
//
// Bound: HBM, 2 bytes read and 1 written per value (and the other way round); a warp takes 1024 columns of a row with all its
// 16-byte loads in flight, eight neighbouring rows share a block so that their 4-byte scales fill whole sectors. In bf16 32768 x 4096 takes
// 64 us there (6.3 TB/s) and 68 back (6.0).
#include "fp8_rows.cuh"

namespace {

constexpr int Q_ROWS = 8;          // rows (warps) of a block
constexpr int Q_COLS = 1024;       // columns of a warp: four vectors of eight values for every lane

template <typename T, bool VEC>
__global__ void __launch_bounds__(Q_ROWS * 32)
    fp8_quantize_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q, long long ldq, float* __restrict__ s,
                             long long lds, long long rows, int K) {
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * Q_ROWS + (threadIdx.x >> 5);
  const int c0 = blockIdx.y * Q_COLS;
  pdl_launch_dependents();                       // a product of these rows may set itself up meanwhile
  if (row >= rows) return;                       // whole warps
  const T* xr = x + row * ldx;
  Eight<T> v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = c0 + i * 256 + lane * 8;
    if (VEC && c < K) v[i].load(xr + c);
    else v[i].load_some(xr + c, VEC ? 0 : K - c);
  }
  uint2 w[4];
  int e[4];
  codes4(v, w, e);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = c0 + i * 256 + lane * 8;
    // rows of codes start on 16 bytes and are padded to them, so a vector that begins inside a row ends inside its padding
    if (c < K) *reinterpret_cast<uint2*>(q + row * ldq + c) = w[i];
    if ((lane & 15) == 0 && c < K) s[(long long)(c >> 7) * lds + row] = __uint_as_float((uint32_t)e[i] << 23);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(Q_ROWS * 32)
    fp8_dequantize_rows_kernel(const uint8_t* __restrict__ q, long long ldq, const float* __restrict__ s, long long lds,
                               T* __restrict__ x, long long ldx, long long rows, int K) {
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * Q_ROWS + (threadIdx.x >> 5);
  const int c0 = blockIdx.y * Q_COLS;
  if (row >= rows) return;
  uint2 raw[4];
  float sc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = c0 + i * 256 + lane * 8;
    raw[i] = make_uint2(0u, 0u);
    sc[i] = 0.f;
    if (c < K) {
      if (VEC || c + 8 <= K) {
        raw[i] = __ldg(reinterpret_cast<const uint2*>(q + row * ldq + c));
      } else {
        for (int j = 0; c + j < K; ++j) (j < 4 ? raw[i].x : raw[i].y) |= (uint32_t)q[row * ldq + c + j] << (8 * (j & 3));
      }
      sc[i] = __ldg(s + (long long)(c >> 7) * lds + row);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = c0 + i * 256 + lane * 8;
    if (c >= K) break;
    alignas(16) T o[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_fp8x2_storage_t two = (__nv_fp8x2_storage_t)((j < 2 ? raw[i].x : raw[i].y) >> (16 * (j & 1)));
      const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
      put2(o + 2 * j, make_float2(f.x * sc[i], f.y * sc[i]));
    }
    T* xr = x + row * ldx + c;
    if (VEC) {
#pragma unroll
      for (int h = 0; h < (int)(sizeof(T) * 8 / 16); ++h) reinterpret_cast<uint4*>(xr)[h] = reinterpret_cast<const uint4*>(o)[h];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < K) xr[j] = o[j];
    }
  }
}

// Rows of x that start on 16 bytes and are whole vectors. Without the ends of a row in the loops 32768 x 4096 takes 68 us back, 74 with them.
bool whole_vectors(const void* p, long long ld, int size, int K) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * size) % 16 == 0 && K % 8 == 0;
}

template <typename T>
int launch_quantize(const void* x, long long ldx, void* q, long long ldq, float* s, long long lds, long long rows, int K, cudaStream_t st) {
  const dim3 grid((unsigned)((rows + Q_ROWS - 1) / Q_ROWS), (unsigned)((K + Q_COLS - 1) / Q_COLS));
  if (whole_vectors(x, ldx, sizeof(T), K))
    fp8_quantize_rows_kernel<T, true><<<grid, Q_ROWS * 32, 0, st>>>((const T*)x, ldx, (uint8_t*)q, ldq, s, lds, rows, K);
  else
    fp8_quantize_rows_kernel<T, false><<<grid, Q_ROWS * 32, 0, st>>>((const T*)x, ldx, (uint8_t*)q, ldq, s, lds, rows, K);
  return (int)cudaGetLastError();
}

template <typename T>
int launch_dequantize(const void* q, long long ldq, const float* s, long long lds, void* x, long long ldx, long long rows, int K,
                      cudaStream_t st) {
  const dim3 grid((unsigned)((rows + Q_ROWS - 1) / Q_ROWS), (unsigned)((K + Q_COLS - 1) / Q_COLS));
  if (whole_vectors(x, ldx, sizeof(T), K))
    fp8_dequantize_rows_kernel<T, true><<<grid, Q_ROWS * 32, 0, st>>>((const uint8_t*)q, ldq, s, lds, (T*)x, ldx, rows, K);
  else
    fp8_dequantize_rows_kernel<T, false><<<grid, Q_ROWS * 32, 0, st>>>((const uint8_t*)q, ldq, s, lds, (T*)x, ldx, rows, K);
  return (int)cudaGetLastError();
}

bool bad_rows(const void* q, long long ldq, long long lds, long long rows, int K) {
  return rows > (1ll << 33) || K > (1 << 26) || (reinterpret_cast<uintptr_t>(q) & 15) || (ldq & 15) || ldq < K || lds < rows;
}

}  // namespace

// x [rows, K] with row stride ldx (elements); dtype 0: bf16, 1: fp16, 2: fp32. q: codes, rows of ldq bytes (a multiple of 16, on 16
// bytes); s: fp32 [ceil(K / 128)][lds], lds >= rows.
extern "C" int axb_fp8_quantize_rows(const void* x, long long ldx, int dtype, void* q, long long ldq, float* s, long long lds,
                                     long long rows, int K, void* stream) {
  if (rows <= 0 || K <= 0) return 0;
  if (bad_rows(q, ldq, lds, rows, K)) return -2;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case 0: return launch_quantize<__nv_bfloat16>(x, ldx, q, ldq, s, lds, rows, K, st);
    case 1: return launch_quantize<__half>(x, ldx, q, ldq, s, lds, rows, K, st);
    case 2: return launch_quantize<float>(x, ldx, q, ldq, s, lds, rows, K, st);
    default: return -2;
  }
}

extern "C" int axb_fp8_dequantize_rows(const void* q, long long ldq, const float* s, long long lds, void* x, long long ldx, int dtype,
                                       long long rows, int K, void* stream) {
  if (rows <= 0 || K <= 0) return 0;
  if (bad_rows(q, ldq, lds, rows, K)) return -2;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case 0: return launch_dequantize<__nv_bfloat16>(q, ldq, s, lds, x, ldx, rows, K, st);
    case 1: return launch_dequantize<__half>(q, ldq, s, lds, x, ldx, rows, K, st);
    case 2: return launch_dequantize<float>(q, ldq, s, lds, x, ldx, rows, K, st);
    default: return -2;
  }
}

// A block of `_pack` (ops/fp8.py): `rows` rows of codes, K rounded up to 16 bytes, and behind them the scales, fp32 [ceil(K / 128)][rows
// rounded up to 4]. One argument: converting ten one by one costs the host as much as a fifth of the launch.
struct AxbFp8Rows {
  void* x;
  void* q;
  void* stream;
  long long ldx, rows;
  int K, dtype;
};
static_assert(sizeof(AxbFp8Rows) == 3 * 8 + 2 * 8 + 2 * 4, "no gaps");

extern "C" int axb_fp8_pack_rows(const AxbFp8Rows* a) {
  const long long ldq = (a->K + 15ll) & ~15ll, lds = (a->rows + 3) & ~3ll;
  float* s = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(a->q) + ldq * a->rows);
  return axb_fp8_quantize_rows(a->x, a->ldx, a->dtype, a->q, ldq, s, lds, a->rows, a->K, a->stream);
}

extern "C" int axb_fp8_unpack_rows(const AxbFp8Rows* a) {
  const long long ldq = (a->K + 15ll) & ~15ll, lds = (a->rows + 3) & ~3ll;
  const float* s = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(a->q) + ldq * a->rows);
  return axb_fp8_dequantize_rows(a->q, ldq, s, lds, a->x, a->ldx, a->dtype, a->rows, a->K, a->stream);
}
