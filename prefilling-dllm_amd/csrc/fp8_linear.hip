// Matrix product with 8-bit floating-point operands (OCP e4m3) and a scale for each block of 128 for gfx950:
//
//   y[m, n] = sum over blocks kb of  sx[m, kb] * sw[n / 128, kb] * sum over k in kb of xq[m, k] * wq[n, k]
//
// One pass of 128 bytes of k is one block: its product is formed by the 32x32x64 matrix instruction from zero and added to
// the fp32 accumulators with its scale.  A lane owns one row m of the result, so the scale is one number per lane, column
// of tiles and block.
//
// Precision.  The instruction multiplies exactly and adds eight products at a time on a grid of 2^-13 of the largest of
// them (measured: beside a product of 2^16 one of 2^3 counts in full, one of 2^2 not at all), then adds the groups in
// fp32.  On random operands that is 1.5e-5 of the result in the root mean square, far below the half step of the bf16
// output (3.9e-3); for that reason the output is bf16 only.

#include "gemm_core.h"

namespace pdllm {

typedef __attribute__((ext_vector_type(8))) int i32x8;

// ---- quantisation --------------------------------------------------------------------------------------------------

// The smallest power of two s with amax / s <= 448 (so that x / s is exact), as its bits; 1 for a block of zeros, NaN for
// one that holds an infinity or a NaN (the rows it takes part in come out NaN).  amax as the bits of |x|.
__device__ __forceinline__ unsigned block_scale_bits(unsigned amax) {
  if (amax >= 0x7f800000u) return 0x7fc00000u;
  if (amax == 0) return 0x3f800000u;
  const int e = (int)(amax >> 23) - ((amax & 0x7fffffu) > 0x600000u ? 7 : 8);  // 448 = 1.75 * 2^8
  return (unsigned)(e < 1 ? 1 : e) << 23;
}
// 1 / s of a power of two; 0 for NaN
__device__ __forceinline__ float inverse_scale(unsigned s) {
  return s >= 0x7f800000u ? 0.f : __uint_as_float((254u << 23) - s);
}
__device__ __forceinline__ unsigned max_bits(const uint4& v) {
  unsigned m = 0;
  const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned lo = (w[i] & 0x7fffu) << 16, hi = w[i] & 0x7fff0000u;
    m = m > lo ? m : lo;
    m = m > hi ? m : hi;
  }
  return m;
}
// eight bf16 values times inv as e4m3 (round to nearest even)
__device__ __forceinline__ uint2 to_e4m3(const uint4& v, float inv) {
  const unsigned w[4] = {v.x, v.y, v.z, v.w};
  unsigned r[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int q = __builtin_amdgcn_cvt_pk_fp8_f32(bf16_bits_to_f32(w[2 * i] & 0xffffu) * inv, bf16_bits_to_f32(w[2 * i] >> 16) * inv, 0, false);
    q = __builtin_amdgcn_cvt_pk_fp8_f32(bf16_bits_to_f32(w[2 * i + 1] & 0xffffu) * inv, bf16_bits_to_f32(w[2 * i + 1] >> 16) * inv, q, true);
    r[i] = (unsigned)q;
  }
  return make_uint2(r[0], r[1]);
}

// One scale for each row and 128 columns; 16 lanes to a block.  HBM-bound: 2 bytes read and 1 written per value.
__global__ __launch_bounds__(256) void fp8_quantize_rows_kernel(const char* __restrict__ x, long x_stride, long M, int K,
                                                                char* __restrict__ q, long q_stride, float* __restrict__ scale,
                                                                long s_row, long s_blk) {
  const int kb = (K + 127) / 128;
  const long id = ((long)blockIdx.x * 256 + threadIdx.x) >> 4;
  const long row = id / kb;
  const int b = (int)(id - row * kb);
  if (row >= M) return;  // (the 16 lanes of a block leave together)
  const int k = b * 128 + (threadIdx.x & 15) * 8;
  uint4 v = {0, 0, 0, 0};
  if (k < K) v = *reinterpret_cast<const uint4*>(x + row * x_stride + 2L * k);
  unsigned m = max_bits(v);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    const unsigned t = __shfl_xor(m, o, 64);
    m = m > t ? m : t;
  }
  const unsigned s = block_scale_bits(m);
  if (k < K) *reinterpret_cast<uint2*>(q + row * q_stride + k) = to_e4m3(v, inverse_scale(s));
  if ((threadIdx.x & 15) == 0) scale[row * s_row + b * s_blk] = __uint_as_float(s);
}

// One scale for each block of 128 x 128 of a weight; one workgroup per block, the block in registers between the two steps.
__global__ __launch_bounds__(256) void fp8_quantize_blocks_kernel(const char* __restrict__ w, long w_stride, long N, int K,
                                                                  char* __restrict__ q, long q_stride, float* __restrict__ scale,
                                                                  long s_row, long s_blk) {
  __shared__ unsigned sh[4];
  const int kb = (K + 127) / 128;
  const long rb = blockIdx.x / kb;
  const int b = (int)(blockIdx.x - rb * kb);
  const int k = b * 128 + (threadIdx.x & 15) * 8;
  uint4 v[8];
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long row = rb * 128 + 16 * i + (threadIdx.x >> 4);
    v[i] = make_uint4(0, 0, 0, 0);
    if (row < N && k < K) v[i] = *reinterpret_cast<const uint4*>(w + row * w_stride + 2L * k);
    const unsigned t = max_bits(v[i]);
    m = m > t ? m : t;
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned t = __shfl_xor(m, o, 64);
    m = m > t ? m : t;
  }
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) m = m > sh[i] ? m : sh[i];
  const unsigned s = block_scale_bits(m);
  const float inv = inverse_scale(s);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long row = rb * 128 + 16 * i + (threadIdx.x >> 4);
    if (row < N && k < K) *reinterpret_cast<uint2*>(q + row * q_stride + k) = to_e4m3(v[i], inv);
  }
  if (threadIdx.x == 0) scale[rb * s_row + b * s_blk] = __uint_as_float(s);
}

// ---- the product ---------------------------------------------------------------------------------------------------

struct Fp8Params {
  const char* x;  // [M, K] e4m3
  const char* w;  // [N, K]
  const float* sx;
  const float* sw;
  long x_stride, w_stride;              // bytes
  long sx_row, sx_blk, sw_row, sw_blk;  // elements
  long M, N;
  int K;
  __bf16* out;
  long o_stride;  // elements
  int vec;        // rows of the output are 8-byte aligned
  int m_tiles, n_tiles;  // tiles of output features, of rows
};

template <class T>
__device__ __forceinline__ void fp8_tile(const Fp8Params& p, char* lds) {
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / T::WN, wn = wave % T::WN;
  const unsigned lds_base = (unsigned)(size_t)lds;
  const int id = xcd_remap(blockIdx.x, gridDim.x);
  const int per = 4 * p.m_tiles;  // four neighbouring row tiles share a strip of the weight in one L2
  const int g = id / per;
  const int left = p.n_tiles - 4 * g;
  const int width = left < 4 ? left : 4;
  const int r = id - g * per;
  const int mt = __builtin_amdgcn_readfirstlane(r / width);
  const int nt = __builtin_amdgcn_readfirstlane(4 * g + r - r / width * width);

  const long f0 = (long)mt * T::TM, r0 = (long)nt * T::TN;
  LoadKC<T::LA> la;
  la.init(p.w + f0 * p.w_stride, p.N - f0, (unsigned)p.w_stride, (unsigned)p.K, wave, lane);
  LoadKC<T::LB> lb;
  lb.init(p.x + r0 * p.x_stride, p.M - r0, (unsigned)p.x_stride, (unsigned)p.K, wave, lane);
  auto issue = [&](int t, unsigned dst) __attribute__((always_inline)) {
    la.issue(t, dst + wave * (T::LA * 1024));
    lb.issue(t, dst + T::A_BYTES + wave * (T::LB * 1024));
  };
  // scales: the wave's features lie in one block of 128
  const long fw = f0 + wm * (32 * T::MT);
  const long fb = fw < p.N ? fw / 128 : (p.N - 1) / 128;
  const float* sw = p.sw + fb * p.sw_row;
  const float* sx[T::NT];
#pragma unroll
  for (int j = 0; j < T::NT; ++j) {
    const long row = r0 + (wn * T::NT + j) * 32 + l32;
    sx[j] = p.sx + (row < p.M ? row : p.M - 1) * p.sx_row;
  }

  Frag<T::MT, false, T::TM> fa;
  Frag<T::NT, false, T::TN> fb_;
  fa.init(lds_base, wm * T::MT * 32, lane);
  fb_.init(lds_base + T::A_BYTES, wn * T::NT * 32, lane);
  f32x16 acc[T::MT][T::NT];
#pragma unroll
  for (int i = 0; i < T::MT; ++i)
#pragma unroll
    for (int j = 0; j < T::NT; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  const int steps = (p.K + 127) / 128;
  float sc[T::NT], sn[T::NT];
  {
    const float w0 = sw[0];
#pragma unroll
    for (int j = 0; j < T::NT; ++j) sn[j] = sx[j][0] * w0;
  }
#pragma unroll
  for (int s = 0; s < T::ST - 1; ++s)
    if (s < steps) issue(s, lds_base + s * T::STAGE);
  unsigned cur = 0, nxt = (T::ST - 1) * T::STAGE;
  bf16x8 A[2][4], B[T::NT][4];
  for (int t = 0; t < steps; ++t) {
    if (T::ST > 2 && t + T::ST - 2 < steps) vm_wait<(T::ST - 2) * (T::LA + T::LB)>();
    else vm_wait<0>();
    wg_barrier();
    fb_.template read<0, 0>(B[0][0], cur);
    fb_.template read<1, 0>(B[0][1], cur);
    fb_.template read<2, 0>(B[0][2], cur);
    fb_.template read<3, 0>(B[0][3], cur);
    if constexpr (T::NT > 1) {
      fb_.template read<0, 1>(B[1][0], cur);
      fb_.template read<1, 1>(B[1][1], cur);
      fb_.template read<2, 1>(B[1][2], cur);
      fb_.template read<3, 1>(B[1][3], cur);
    }
    fa.template read<0, 0>(A[0][0], cur);
    fa.template read<1, 0>(A[0][1], cur);
    fa.template read<2, 0>(A[0][2], cur);
    fa.template read<3, 0>(A[0][3], cur);
#pragma unroll
    for (int j = 0; j < T::NT; ++j) sc[j] = sn[j];
    {
      const int tn = t + 1 < steps ? t + 1 : t;
      const float w1 = sw[tn * p.sw_blk];
#pragma unroll
      for (int j = 0; j < T::NT; ++j) sn[j] = sx[j][tn * p.sx_blk] * w1;
    }
    if (t + T::ST - 1 < steps) issue(t + T::ST - 1, lds_base + nxt);
    lgkm_wait<0>();
#pragma unroll
    for (int j = 0; j < T::NT; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) tie(B[j][k]);
#pragma unroll
    for (int i = 0; i < T::MT; ++i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) tie(A[i & 1][k]);
      if (i + 1 < T::MT) {
        auto next = [&](auto jt) __attribute__((always_inline)) {
          constexpr int J = decltype(jt)::value;
          fa.template read<0, J>(A[(i + 1) & 1][0], cur);
          fa.template read<1, J>(A[(i + 1) & 1][1], cur);
          fa.template read<2, J>(A[(i + 1) & 1][2], cur);
          fa.template read<3, J>(A[(i + 1) & 1][3], cur);
        };
        if (i == 0) next(std::integral_constant<int, (T::MT > 1 ? 1 : 0)>{});
        else if (i == 1) next(std::integral_constant<int, (T::MT > 2 ? 2 : 0)>{});
        else next(std::integral_constant<int, (T::MT > 3 ? 3 : 0)>{});
      }
      f32x16 zero;
#pragma unroll
      for (int e = 0; e < 16; ++e) zero[e] = 0.f;
      auto pair = [](const bf16x8& a, const bf16x8& b) __attribute__((always_inline)) {
        typedef __attribute__((ext_vector_type(4))) int i32x4;
        return __builtin_shufflevector(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), 0, 1, 2, 3, 4, 5, 6, 7);
      };
#pragma unroll
      for (int j = 0; j < T::NT; ++j) {
        f32x16 d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(pair(A[i & 1][0], A[i & 1][1]), pair(B[j][0], B[j][1]), zero,
                                                                   0, 0, 0, 0, 0, 0);
        d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(pair(A[i & 1][2], A[i & 1][3]), pair(B[j][2], B[j][3]), d, 0, 0, 0,
                                                            0, 0, 0);
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = __builtin_fmaf(d[e], sc[j], acc[i][j][e]);
      }
      if (i + 1 < T::MT) lgkm_wait<0>();
    }
    cur = cur == (T::ST - 1) * T::STAGE ? 0u : cur + T::STAGE;
    nxt = nxt == (T::ST - 1) * T::STAGE ? 0u : nxt + T::STAGE;
  }

#pragma unroll
  for (int j = 0; j < T::NT; ++j) {
    const long row = r0 + (wn * T::NT + j) * 32 + l32;
    if (row >= p.M) continue;
#pragma unroll
    for (int i = 0; i < T::MT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const long f = fw + 32 * i + 8 * q + 4 * h;
        if (f >= p.N) continue;
        const long o = row * p.o_stride + f;
        if (p.vec && f + 4 <= p.N) {
          const uint2 v = {pack_bf16x2(acc[i][j][4 * q], acc[i][j][4 * q + 1]),
                           pack_bf16x2(acc[i][j][4 * q + 2], acc[i][j][4 * q + 3])};
          *reinterpret_cast<uint2*>(p.out + o) = v;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (f + e < p.N) p.out[o + e] = (__bf16)acc[i][j][4 * q + e];
        }
      }
  }
}

// (a function of its own: the host compiler cannot emit a kernel whose lambda holds a buffer descriptor)
template <class T>
__global__ __launch_bounds__(T::THREADS, 2) void fp8_linear_kernel(const Fp8Params p) {
  __shared__ __attribute__((aligned(1024))) char lds[T::LDS];
  fp8_tile<T>(p, lds);
}

namespace {

using TileL = Tile<4, 2, 2, 4, 2>;   // 256 features x 256 rows, 8 waves
using TileM = Tile<2, 2, 4, 2, 3>;   // 256 x 128
using TileS2 = Tile<1, 2, 4, 1, 3>;  // 128 x 64, 4 waves
using TileS = Tile<1, 1, 4, 1, 4>;   // 128 x 32

constexpr long kMaxRows = 1L << 24;

template <class T>
int launch_fp8(Fp8Params& p, hipStream_t s) {
  p.m_tiles = (int)((p.N + T::TM - 1) / T::TM);
  p.n_tiles = (int)((p.M + T::TN - 1) / T::TN);
  const long grid = (long)p.m_tiles * p.n_tiles;
  if (grid > 0x7fffffffL) return PDLLM_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(fp8_linear_kernel<T>, dim3((unsigned)grid), dim3(T::THREADS), 0, s, p);
  return launch_status();
}

int check_quantize(const void* x, int64_t x_stride, int64_t rows, int32_t K, const void* q, int64_t q_stride, const void* scale,
                   int64_t s_row, int64_t s_blk) {
  if (rows < 0 || K <= 0 || K % 16 || K > (1 << 20) || rows > (1L << 30)) return PDLLM_ERR_SHAPE;
  if (rows == 0) return PDLLM_OK;
  if (!x || !q || !scale) return PDLLM_ERR_NULL;
  if (x_stride < K || x_stride % 8 || q_stride < K || q_stride % 16 || (uintptr_t)x % 16 || (uintptr_t)q % 16 ||
      (uintptr_t)scale % 4 || s_row < 0 || s_blk < 0)
    return PDLLM_ERR_STRIDE;
  return PDLLM_OK;
}

}  // namespace

}  // namespace pdllm

using namespace pdllm;

extern "C" int pdllm_fp8_quantize_rows(const void* x, int64_t x_stride, int64_t n_rows, int32_t k, void* q, int64_t q_stride,
                                       float* scale, int64_t scale_row_stride, int64_t scale_block_stride,
                                       pdllm_stream_t stream) {
  const int st = check_quantize(x, x_stride, n_rows, k, q, q_stride, scale, scale_row_stride, scale_block_stride);
  if (st != PDLLM_OK || n_rows == 0) return st;
  const long blocks = n_rows * ((k + 127) / 128);
  if ((blocks + 15) / 16 > 0x7fffffffL) return PDLLM_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(fp8_quantize_rows_kernel, dim3((unsigned)((blocks + 15) / 16)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), static_cast<const char*>(x), 2L * x_stride, (long)n_rows, k,
                     static_cast<char*>(q), (long)q_stride, scale, (long)scale_row_stride, (long)scale_block_stride);
  return launch_status();
}

extern "C" int pdllm_fp8_quantize_blocks(const void* w, int64_t w_stride, int64_t n_rows, int32_t k, void* q, int64_t q_stride,
                                         float* scale, int64_t scale_row_stride, int64_t scale_block_stride,
                                         pdllm_stream_t stream) {
  const int st = check_quantize(w, w_stride, n_rows, k, q, q_stride, scale, scale_row_stride, scale_block_stride);
  if (st != PDLLM_OK || n_rows == 0) return st;
  const long blocks = (n_rows + 127) / 128 * ((k + 127) / 128);
  if (blocks > 0x7fffffffL) return PDLLM_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(fp8_quantize_blocks_kernel, dim3((unsigned)blocks), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const char*>(w), 2L * w_stride, (long)n_rows, k, static_cast<char*>(q), (long)q_stride, scale,
                     (long)scale_row_stride, (long)scale_block_stride);
  return launch_status();
}

extern "C" int pdllm_fp8_linear(const void* x, int64_t x_stride, const float* x_scale, int64_t x_scale_row_stride,
                                int64_t x_scale_block_stride, const void* weight, int64_t weight_stride,
                                const float* weight_scale, int64_t weight_scale_row_stride,
                                int64_t weight_scale_block_stride, int64_t m, int64_t n, int32_t k, void* out,
                                int64_t out_stride, pdllm_stream_t stream) {
  if (m < 0 || n <= 0 || k <= 0 || k % 16 || k > (1 << 20) || m > kMaxRows || n > (1L << 30)) return PDLLM_ERR_SHAPE;
  if (m == 0) return PDLLM_OK;
  if (!x || !x_scale || !weight || !weight_scale || !out) return PDLLM_ERR_NULL;
  if (x_stride < k || x_stride % 16 || weight_stride < k || weight_stride % 16 || (uintptr_t)x % 16 || (uintptr_t)weight % 16 ||
      x_stride * 256 >= 0x7fffffffL || weight_stride * 256 >= 0x7fffffffL || out_stride < n || x_scale_row_stride < 0 ||
      x_scale_block_stride < 0 || weight_scale_row_stride < 0 || weight_scale_block_stride < 0 ||
      (uintptr_t)out % 2)
    return PDLLM_ERR_STRIDE;
  Fp8Params p = {};
  p.x = static_cast<const char*>(x);
  p.w = static_cast<const char*>(weight);
  p.sx = x_scale;
  p.sw = weight_scale;
  p.x_stride = x_stride;
  p.w_stride = weight_stride;
  p.sx_row = x_scale_row_stride;
  p.sx_blk = x_scale_block_stride;
  p.sw_row = weight_scale_row_stride;
  p.sw_blk = weight_scale_block_stride;
  p.M = m;
  p.N = n;
  p.K = k;
  p.out = static_cast<__bf16*>(out);
  p.o_stride = out_stride;
  p.vec = out_stride % 4 == 0 && (uintptr_t)out % 8 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (m <= 32) return launch_fp8<TileS>(p, s);
  if (m <= 64) return launch_fp8<TileS2>(p, s);
  if (m <= 128) return launch_fp8<TileM>(p, s);
  return launch_fp8<TileL>(p, s);
}
