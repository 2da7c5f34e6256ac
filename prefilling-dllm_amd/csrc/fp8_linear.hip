// Matrix product with 8-bit floating-point operands (OCP e4m3) and a scale for each block of 128 for gfx950:
//
//   y[m, n] = sum over blocks kb of  sx[m, kb] * sw[n / 128, kb] * sum over k in kb of xq[m, k] * wq[n, k]
//
// One pass of 128 bytes of k is one block: its product is formed by one 16x16x128 matrix instruction from zero and added to
// the fp32 accumulators with its scale.  A lane owns one row m of the result, so the scale is one number per lane, column
// of tiles and block.  (From registers, with normally distributed values, 16x16x128 sustains 4430 TFLOP/s at the card's power limit,
// 32x32x64 4020.)
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

// One scale for each row and 128 columns; 16 lanes to a block, 16 blocks of a row to a workgroup.  HBM-bound: 2 bytes read and 1
// written per value (8200 x 3584: 16 us called in a row, 5.5 TB/s; 18 to 24 in front of a product).
__global__ __launch_bounds__(256) void fp8_quantize_rows_kernel(const char* __restrict__ x, long x_stride, int groups, int K,
                                                                char* __restrict__ q, long q_stride, float* __restrict__ scale,
                                                                long s_row, long s_blk) {
  const unsigned row = blockIdx.x / (unsigned)groups;
  const int b = (int)(blockIdx.x - row * (unsigned)groups) * 16 + (threadIdx.x >> 4);
  const int k = b * 128 + (threadIdx.x & 15) * 8;
  if (b * 128 >= K) return;  // (the 16 lanes of a block leave together)
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

// One scale for each block of 128 x 128 of a weight; one workgroup per block, the block in registers between the two steps.  HBM-bound
// (152064 x 3584: 309 us, 5.3 TB/s; 18944 x 3584: 31 us).
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
  const char* x;  // [M, K] e4m3 (bf16 where a kernel quantises on the way)
  const char* w;  // [N, K]
  const float* sx;
  const float* sw;
  long x_stride, w_stride;              // bytes
  long sx_row, sx_blk, sw_row, sw_blk;  // elements
  long M, N;
  int K;
  __bf16* out;
  long o_stride;  // elements
  int m_tiles, n_tiles;  // tiles of output features, of rows
};

// A wave's operand fragments, blocks of 16 rows: lane 16 g + l holds, of row l, the 16 bytes of k at 16 g and at 64 + 16 g (any order
// that both operands share does).
struct Frag8 {
  unsigned a[2];
  __device__ __forceinline__ void init(unsigned lds_base, int first, int lane) {
    const int l16 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int q = 0; q < 2; ++q) a[q] = lds_base + (first + l16) * KB + (((4 * q + g) ^ kc_xor(l16)) << 4);
  }
  template <int J>
  __device__ __forceinline__ void read(bf16x8 (&d)[2], unsigned stage) const {
    lds_read_b128<J * 16 * KB>(d[0], a[0] + stage);
    lds_read_b128<J * 16 * KB>(d[1], a[1] + stage);
  }
};

// A tile of T::TM features x T::TN rows; bound by the matrix instructions and, for the largest products, the card's power.  The
// tile's whole stage of B stays in registers, blocks of A pass by; each product waits two instructions before it is added, and reads
// of the next block, and copies of the stages behind, go between the instructions (8200 rows x 18944 x 3584: 541 us with
// 32x32x64 instructions, reads and copies in front of them; 489 us so, 2.27 PFLOP/s.  2048 x 8192 x 8192: 109 us, 2.52 PFLOP/s).
template <class T>
__device__ __forceinline__ void fp8_tile(const Fp8Params& p, char* lds) {
  const int lane = threadIdx.x & 63, l16 = lane & 15;
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
  auto issue = [&](int t, unsigned dst, auto copy) __attribute__((always_inline)) {
    constexpr int I = decltype(copy)::value;
    if constexpr (I < T::LA) la.template one<I>(t, dst + wave * (T::LA * 1024));
    else lb.template one<I - T::LA>(t, dst + T::A_BYTES + wave * (T::LB * 1024));
  };
  // scales: the wave's features lie in one block of 128
  const long fw = f0 + wm * (32 * T::MT);
  const long fb = fw < p.N ? fw / 128 : (p.N - 1) / 128;
  const float* sw = p.sw + fb * p.sw_row;
  const float* sx = p.sx + r0 * p.sx_row;
  constexpr int NI = 2 * T::MT, NJ = 2 * T::NT;  // blocks of 16 features, of 16 rows
  unsigned sx_off[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int row = wn * (32 * T::NT) + 16 * j + l16;
    sx_off[j] = (unsigned)(r0 + row < p.M ? row : (int)(p.M - 1 - r0)) * (unsigned)p.sx_row;
  }

  Frag8 fa, fb_;
  fa.init(lds_base, wm * T::MT * 32, lane);
  fb_.init(lds_base + T::A_BYTES, wn * T::NT * 32, lane);
  Acc<T> acc;
  acc.clear();
  const int steps = (p.K + 127) / 128;
  constexpr int COPIES = T::LA + T::LB, HALF = COPIES / 2;
  // The scales of a stage are fetched ST - 1 stages ahead, right in front of the copies of the stage behind it: loads return in
  // order, so waiting for them never waits for copies that are not needed yet.
  constexpr int AHEAD = T::ST - 1;
  float sc[NJ], qx[AHEAD][NJ], qw[AHEAD];
  auto fetch = [&](int t, float (&x)[NJ], float& w) __attribute__((always_inline)) {
    t = t < steps ? t : steps - 1;
    w = sw[t * p.sw_blk];
#pragma unroll
    for (int j = 0; j < NJ; ++j) x[j] = (sx + t * p.sx_blk)[sx_off[j]];
  };
#pragma unroll
  for (int a = 0; a < AHEAD; ++a) fetch(a, qx[a], qw[a]);
  // Copies of stages behind the last one read nothing: no branches in the loop.  The second half of stage ST - 1 follows in the
  // first stage.
  unrolled<T::ST * COPIES - (COPIES - HALF)>([&](auto n) __attribute__((always_inline)) {
    constexpr int s = decltype(n)::value / COPIES;
    issue(s, lds_base + s * T::STAGE, std::integral_constant<int, decltype(n)::value % COPIES>{});
  });
  vm_wait<(T::ST - 2) * COPIES + HALF>();
  wg_barrier();
  unsigned cur = 0, old = (T::ST - 1) * T::STAGE;
  bf16x8 A[2][2], B[NJ][2];  // A: this block and the next
  unrolled<NJ>([&](auto j) __attribute__((always_inline)) { fb_.template read<decltype(j)::value>(B[decltype(j)::value], cur); });
  fa.template read<0>(A[0], cur);
  auto whole = [](const bf16x8 (&a)[2]) __attribute__((always_inline)) {
    typedef __attribute__((ext_vector_type(4))) int i32x4;
    return __builtin_shufflevector(__builtin_bit_cast(i32x4, a[0]), __builtin_bit_cast(i32x4, a[1]), 0, 1, 2, 3, 4, 5, 6, 7);
  };
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  int t = 0;
  do {
    // Blocks of 16 features in turn.  The products of a block of 16 x 16 are added to the accumulators behind the matrix
    // instruction after the next one, so that the additions never wait for their result.
    f32x4 d[3];
    auto add = [&](auto n_tag) __attribute__((always_inline)) {
      constexpr int n = decltype(n_tag)::value;
      if constexpr (n >= 0) {
        f32x4& to = acc.v[n / NJ][n % NJ];
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = __builtin_fmaf(d[n % 3][e], sc[n % NJ], to[e]);
        // (pinned here: moved behind the loop's end, the additions would keep the products of a whole stage alive)
        asm volatile("" : "+v"(to));
      }
    };
    unrolled<NI>([&](auto block) __attribute__((always_inline)) {
      constexpr int i = decltype(block)::value;
      lgkm_wait<0>();
      tie(A[i & 1][0]);
      tie(A[i & 1][1]);
      if constexpr (i == 0) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          tie(B[j][0]);
          tie(B[j][1]);
          sc[j] = qx[0][j] * qw[0];
#pragma unroll
          for (int a = 0; a + 1 < AHEAD; ++a) qx[a][j] = qx[a + 1][j];
        }
#pragma unroll
        for (int a = 0; a + 1 < AHEAD; ++a) qw[a] = qw[a + 1];
      }
      if constexpr (i + 1 == NI) {
        // the stage has been read by this wave; behind the barrier by all, and the next one has landed
        vm_wait<(T::ST - 2) * COPIES>();
        wg_barrier();
        fetch(t + AHEAD, qx[AHEAD - 1], qw[AHEAD - 1]);
        old = cur;
        cur = cur == (T::ST - 1) * T::STAGE ? 0u : cur + T::STAGE;
      }
      unrolled<NJ>([&](auto row) __attribute__((always_inline)) {
        constexpr int j = decltype(row)::value, n = i * NJ + j;
        __builtin_amdgcn_sched_barrier(0);
        d[n % 3] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(whole(A[i & 1]), whole(B[j]), zero, 0, 0, 0, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        // (behind the last stage: reads of whatever the buffer holds, which nothing uses)
        if constexpr (j == 0) fa.template read<(i + 1) % NI>(A[(i + 1) & 1], cur);
        if constexpr (i + 1 == NI) fb_.template read<j>(B[j], cur);
        unrolled<COPIES>([&](auto copy) __attribute__((always_inline)) {
          constexpr int c = decltype(copy)::value;
          if constexpr (c < HALF && i + 1 == NI && c * NJ / HALF == j) issue(t + T::ST, lds_base + old, copy);
          if constexpr (c >= HALF && i == 0 && (c - HALF) * NJ / (COPIES - HALF) == j) issue(t + T::ST - 1, lds_base + old, copy);
        });
        add(std::integral_constant<int, n - 2>{});
      });
    });
    add(std::integral_constant<int, NI * NJ - 2>{});
    add(std::integral_constant<int, NI * NJ - 1>{});
  } while (++t < steps);
  lgkm_wait<0>();
  tie(A[0][0]);
  tie(A[0][1]);
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    tie(B[j][0]);
    tie(B[j][1]);
  }
  vm_wait<0>();

  store_acc<T>(lds, acc, [](float a, float b) __attribute__((always_inline)) { return pack_bf16x2(a, b); }, p.out + r0 * p.o_stride + f0,
               p.o_stride, p.M - r0, p.N - f0);
}

// (a function of its own: the host compiler cannot emit a kernel whose lambda holds a buffer descriptor)
template <class T>
__global__ __launch_bounds__(T::THREADS, 2) void fp8_linear_kernel(const Fp8Params p) {
  __shared__ __attribute__((aligned(1024))) char lds[T::LDS];
  fp8_tile<T>(p, lds);
}

// Up to 32 rows: the weight is read once, straight into registers, and the call waits for memory.  A workgroup takes FT = 16 or
// 32 features and all rows (more rows: 32 of them); its eight waves take every eighth block of k, so that all of the
// workgroup's weight (FT x K bytes) is on its way at once, and their fp32 sums meet in LDS, added in wave order.  16x16x128
// instruction: lane l holds row l & 15 of an operand, bytes 16 (l >> 4) .. + 15 of each half of the block (any order of k that
// both operands share).  1 row x 152064 x 3584: 88 us, 6.2 TB/s; 1 x 4096 x 4096: 5.0 us with an
// e4m3 row and 6.6 to 7.2 with a bf16 row, which is quantised first; the weight's 16.8 MB are 3.4.
template <int FT, int TT, bool BF>
__global__ __launch_bounds__(512, 4) void fp8_stream_kernel(const Fp8Params p) {
  constexpr int NF = FT / 16, U = 2;  // U blocks of a wave in flight
  __shared__ float part[8][TT * 16][FT + 1];
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long f0 = (long)blockIdx.x * FT;
  const long nf = p.N - f0 < FT ? p.N - f0 : FT;
  const long r0 = 16L * TT * blockIdx.y;  // first row of the workgroup's
  const int m = p.M - r0 < 16 * TT ? (int)(p.M - r0) : 16 * TT;
  const __amdgpu_buffer_rsrc_t wr = make_rsrc(p.w + f0 * p.w_stride, (unsigned)((nf - 1) * p.w_stride) + (unsigned)p.K);
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(p.x + r0 * p.x_stride, (unsigned)((m - 1) * p.x_stride) + (unsigned)(BF ? 2 * p.K : p.K));
  unsigned wo[NF], xo[TT], so[TT];
#pragma unroll
  for (int f = 0; f < NF; ++f) wo[f] = f * 16 + l16 < nf ? (unsigned)(f * 16 + l16) * (unsigned)p.w_stride : kOutOfRange;
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int row = t * 16 + l16;
    xo[t] = row < m ? (unsigned)row * (unsigned)p.x_stride : kOutOfRange;
    so[t] = (unsigned)(row < m ? row : m - 1) * (unsigned)p.sx_row;
  }
  const float* sw = p.sw + f0 / 128 * p.sw_row;
  const float* sx = BF ? nullptr : p.sx + r0 * p.sx_row;
  f32x4 acc[NF][TT];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int blocks = (p.K + 127) / 128;
  typedef __attribute__((ext_vector_type(4))) int i32x4;
  auto load = [&](const __amdgpu_buffer_rsrc_t& rs, unsigned row, int kb) __attribute__((always_inline)) {
    const unsigned k0 = kb * 128 + 16 * g, k1 = k0 + 64;
    const i32x4 a = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, k0 < (unsigned)p.K ? row + k0 : kOutOfRange, 0, 0));
    const i32x4 b = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, k1 < (unsigned)p.K ? row + k1 : kOutOfRange, 0, 0));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // bf16 rows: a lane's 32 values of the block, the block's scale from the four lanes that share it
  auto load_quantized = [&](unsigned row, int kb, float& scale) __attribute__((always_inline)) {
    uint4 v[4];
    unsigned amax = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const unsigned k = kb * 128 + (c >> 1) * 64 + 16 * g + (c & 1) * 8;
      v[c] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(xr, k < (unsigned)p.K ? row + 2 * k : kOutOfRange, 0, 0));
      const unsigned b = max_bits(v[c]);
      amax = amax > b ? amax : b;
    }
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) {
      const unsigned b = __shfl_xor(amax, o, 64);
      amax = amax > b ? amax : b;
    }
    const unsigned sb = block_scale_bits(amax);
    scale = __uint_as_float(sb);
    const float inv = inverse_scale(sb);
    i32x8 r;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint2 q = to_e4m3(v[c], inv);
      r[2 * c] = (int)q.x;
      r[2 * c + 1] = (int)q.y;
    }
    return r;
  };
  for (int b0 = wave; b0 < blocks; b0 += 8 * U) {
    i32x8 w[U][NF], x[U][TT];
    float s[U][TT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = b0 + 8 * u;  // (behind the last block: zeros)
#pragma unroll
      for (int f = 0; f < NF; ++f) w[u][f] = load(wr, wo[f], kb);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = b0 + 8 * u;
      const int ks = kb < blocks ? kb : b0;
      const float ws = sw[ks * p.sw_blk];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        if constexpr (BF) {
          x[u][t] = load_quantized(xo[t], kb, s[u][t]);
          s[u][t] = kb < blocks ? s[u][t] * ws : 0.f;
        } else {
          x[u][t] = load(xr, xo[t], kb);
          s[u][t] = kb < blocks ? (sx + ks * p.sx_blk)[so[t]] * ws : 0.f;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          const f32x4 d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[u][f], x[u][t], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[f][t][e] = __builtin_fmaf(d[e], s[u][t], acc[f][t][e]);
        }
  }
  // lane l of a 16x16 result holds column (row of the output) l & 15, rows (features) 4 (l >> 4) .. + 3
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[wave][t * 16 + l16][f * 16 + 4 * g + e] = acc[f][t][e];
  __syncthreads();
  for (int i = threadIdx.x; i < FT * TT * 16; i += 512) {
    const int f = i % FT, row = i / FT;
    if (row >= m || f >= nf) continue;
    float v = part[0][row][f];
#pragma unroll
    for (int q = 1; q < 8; ++q) v += part[q][row][f];
    p.out[(r0 + row) * p.o_stride + f0 + f] = (__bf16)v;
  }
}

// Up to 32 rows and many features: one workgroup per compute unit stays, the rows and their scales in its LDS (they would
// otherwise be read again for every group of features: twice the weight's bytes, through the same L2), and walks over groups
// of 32 features.  Wave (q, c) takes blocks q, q + 8, ... of k of the 16 features c of the group, so that the group's rows of the
// weight, which lie side by side in memory, are asked for together; a ring of U blocks in registers runs on from group to
// group.  The eight partial sums of a result meet in LDS, added in wave order.  32 rows x 152064 x 3584: 107 us, 5.2 TB/s of weight
// and results.
// Rows in LDS: block kb of row r, chunk c at ((kb * R + r) * 8 + (c ^ (r >> 1 & 7))) * 16: 16 rows of one chunk cover all banks.
constexpr int kResidentPad = 33;
constexpr int kResidentQ = 8;  // waves that share the features' k
template <int R>
constexpr long resident_lds(long blocks, long groups) {
  return blocks * R * 132 + kResidentQ * R * kResidentPad * 4 + blocks * groups * 4;
}
template <int TT, int U, bool BF>
__global__ __launch_bounds__(1024, 4) void fp8_resident_kernel(const Fp8Params p) {
  extern __shared__ __attribute__((aligned(1024))) char xs[];
  constexpr int R = 16 * TT;
  typedef __attribute__((ext_vector_type(4))) int i32x4;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kq = wave % kResidentQ, c = wave / kResidentQ;
  const int m = (int)p.M;
  const int blocks = (p.K + 127) / 128;  // at least kResidentQ
  const int tasks = (int)((p.N + 31) / 32), per = (int)gridDim.x;
  const int first = blockIdx.x;
  float* scales = reinterpret_cast<float*>(xs + blocks * R * 128);
  float* part = scales + blocks * R;                   // [kResidentQ][R][kResidentPad]
  float* wscale = part + kResidentQ * R * kResidentPad;  // [groups of this workgroup][blocks]

  int a_task = first, a_kb = kq;  // the block fetched next
  i32x4 ring[U][2];
  auto fetch = [&](i32x4 (&d)[2]) __attribute__((always_inline)) {
    const long f = 32L * a_task + 16 * c;
    const int nf = a_task < tasks && f < p.N ? (int)(p.N - f < 16 ? p.N - f : 16) : 0;
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(p.w + (nf > 0 ? f : 0) * p.w_stride, nf > 0 ? (unsigned)((nf - 1) * p.w_stride) + (unsigned)p.K : 0u);
    const unsigned row = (unsigned)l16 * (unsigned)p.w_stride;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const unsigned k = a_kb * 128 + 64 * q + 16 * g;
      d[q] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, k < (unsigned)p.K ? row + k : kOutOfRange, 0, 0));
    }
    a_kb += kResidentQ;
    if (a_kb >= blocks) {
      a_kb = kq;
      a_task += per;
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) fetch(ring[u]);
  if constexpr (BF) {
    // bf16 rows: 16 lanes to a block, as the quantising kernel does it; four blocks of a lane are fetched together
    const int l = threadIdx.x & 15, all = blocks * R;
    for (int i0 = threadIdx.x >> 4; i0 < all; i0 += 4 * 64) {
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + 64 * u, r = i % R, k = i / R * 128 + 8 * l;
        v[u] = uint4{0, 0, 0, 0};
        if (i < all && r < m && k < p.K) v[u] = *reinterpret_cast<const uint4*>(p.x + (long)r * p.x_stride + 2 * k);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + 64 * u, r = i % R, kb = i / R;
        unsigned amax = max_bits(v[u]);
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
          const unsigned t = __shfl_xor(amax, o, 64);
          amax = amax > t ? amax : t;
        }
        const unsigned sb = block_scale_bits(amax);
        if (i < all) {
          *reinterpret_cast<uint2*>(xs + (((kb * R + r) * 8 + ((l >> 1) ^ ((r >> 1) & 7))) << 4) + 8 * (l & 1)) = to_e4m3(v[u], inverse_scale(sb));
          if (l == 0) scales[i] = __uint_as_float(sb);
        }
      }
    }
  } else {
    for (int i = threadIdx.x; i < blocks * R * 8; i += 1024) {
      const int ch = i & 7, r = (i >> 3) % R, kb = (i >> 3) / R;
      const int k = kb * 128 + 16 * ch;
      uint4 v = {0, 0, 0, 0};
      if (r < m && k < p.K) v = *reinterpret_cast<const uint4*>(p.x + (long)r * p.x_stride + k);
      *reinterpret_cast<uint4*>(xs + (((kb * R + r) * 8 + (ch ^ ((r >> 1) & 7))) << 4)) = v;
    }
    for (int i = threadIdx.x; i < blocks * R; i += 1024) {
      const int r = i % R, kb = i / R;
      scales[i] = r < m ? p.sx[r * p.sx_row + kb * p.sx_blk] : 0.f;
    }
  }
  const int mine = first < tasks ? (tasks - 1 - first) / per + 1 : 0;
  for (int i = threadIdx.x; i < mine * blocks; i += 1024) {
    const int t = i / blocks;
    wscale[i] = p.sw[((first + t * per) >> 2) * p.sw_row + (i - t * blocks) * p.sw_blk];  // (32 features: within one block)
  }
  __syncthreads();

  f32x4 acc[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int total = mine * ((blocks - kq + kResidentQ - 1) / kResidentQ);
  int task = first, kb = kq;
  const unsigned rd = (unsigned)(l16 * 128);
  const unsigned ch0 = (unsigned)((g ^ ((l16 >> 1) & 7)) << 4), ch1 = (unsigned)(((4 + g) ^ ((l16 >> 1) & 7)) << 4);
  for (int n = 0; n < total; n += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (n + u >= total) break;
      const float ws = wscale[kb];
      const i32x8 w = __builtin_shufflevector(ring[u][0], ring[u][1], 0, 1, 2, 3, 4, 5, 6, 7);
      const char* b = xs + kb * (R * 128) + rd;
      i32x8 x[TT];
      float sc[TT];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const i32x4 x0 = *reinterpret_cast<const i32x4*>(b + t * 2048 + ch0);
        const i32x4 x1 = *reinterpret_cast<const i32x4*>(b + t * 2048 + ch1);
        x[t] = __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
        sc[t] = scales[kb * R + 16 * t + l16];
      }
      f32x4 d[TT];
#pragma unroll
      for (int t = 0; t < TT; ++t) d[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x[t], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = __builtin_fmaf(d[t][e], sc[t] * ws, acc[t][e]);
      fetch(ring[u]);
      kb += kResidentQ;
      if (kb >= blocks) {
        // the group is done: every wave passes these two barriers once per group
        kb = kq;
#pragma unroll
        for (int t = 0; t < TT; ++t) {
#pragma unroll
          for (int e = 0; e < 4; ++e) part[(kq * R + 16 * t + l16) * kResidentPad + 16 * c + 4 * g + e] = acc[t][e];
          acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        lgkm_wait<0>();
        wg_barrier();
        for (int i = threadIdx.x; i < R * 32; i += 1024) {
          const int f = i & 31, row = i >> 5;
          const float* q = part + row * kResidentPad + f;
          float v = q[0];
#pragma unroll
          for (int o = 1; o < kResidentQ; ++o) v += q[o * R * kResidentPad];
          if (row < m && 32L * task + f < p.N) p.out[row * p.o_stride + 32L * task + f] = (__bf16)v;
        }
        lgkm_wait<0>();
        wg_barrier();
        task += per;
        wscale += blocks;
      }
    }
  }
}

namespace {

using TileL = Tile<4, 2, 2, 4, 2>;   // 256 features x 256 rows, 8 waves
using TileM = Tile<2, 2, 4, 2, 3>;   // 256 x 128
using TileS2 = Tile<1, 2, 4, 1, 3>;  // 128 x 64, 4 waves

constexpr long kMaxRows = 1L << 24;

template <class T>
int launch_fp8(Fp8Params& p, hipStream_t s) {
  p.m_tiles = (int)((p.N + T::TM - 1) / T::TM);
  p.n_tiles = (int)((p.M + T::TN - 1) / T::TN);
  const long grid = (long)p.m_tiles * p.n_tiles;
  if (!launch_fits(grid, T::THREADS)) return PDLLM_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(fp8_linear_kernel<T>, dim3((unsigned)grid), dim3(T::THREADS), 0, s, p);
  return launch_status();
}

template <int TT, bool BF>
int launch_resident(Fp8Params& p, hipStream_t s) {
  const long blocks = (p.K + 127) / 128, groups = ((p.N + 31) / 32 + 255) / 256;
  hipLaunchKernelGGL((fp8_resident_kernel<TT, 4, BF>), dim3(256), dim3(1024), (unsigned)resident_lds<16 * TT>(blocks, groups), s, p);
  return launch_status();
}

// 32 features to a workgroup of the streaming kernel read the rows half as often; 16 where 32 would leave compute units idle
bool stream_wide(const Fp8Params& p) { return (p.N + 31) / 32 * ((p.M + 31) / 32) >= 512; }

template <int TT, bool BF>
int launch_stream(Fp8Params& p, hipStream_t s) {
  const bool wide = stream_wide(p);
  const long columns = (p.N + (wide ? 31 : 15)) / (wide ? 32 : 16), rows = (p.M + 16 * TT - 1) / (16 * TT);
  if (!launch_fits(columns, 512) || rows > 65535) return PDLLM_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)columns, (unsigned)rows);
  if (wide) hipLaunchKernelGGL((fp8_stream_kernel<32, TT, BF>), grid, dim3(512), 0, s, p);
  else hipLaunchKernelGGL((fp8_stream_kernel<16, TT, BF>), grid, dim3(512), 0, s, p);
  return launch_status();
}

// Up to 32 rows beside many features: the rows stay in LDS where they fit (K = 3584, 152064 features, us streamed and resident: e4m3
// rows 88 and 90 for 1, 97 and 96 for 8, 110 and 99 for 16, 141 and 107 for 32; bf16 rows, which every streaming workgroup
// quantises again, 122 and 92 for 1, 161 and 102 for 16, 229 and 112 for 32.  16384 features x 4096: 14.8 and 15.8 for 1 row, 16.3
// and 16.1 for 16; 12288 x 2048: 10.8 and 9.7 for 32 rows, 8.2 and 9.2 for 16).
bool resident_fits(const Fp8Params& p, bool bf) {
  const long blocks = (p.K + 127) / 128, groups = ((p.N + 31) / 32 + 255) / 256;
  if (blocks < kResidentQ || p.M > 32) return false;
  if (p.M > 16) return p.N >= 12288 && resident_lds<32>(blocks, groups) <= 160 * 1024;
  return p.N >= 16384 && (bf || p.M > 4) && resident_lds<16>(blocks, groups) <= 160 * 1024;
}

// up to 32 rows
template <bool BF>
int launch_few(Fp8Params& p, hipStream_t s) {
  if (resident_fits(p, BF)) return p.M <= 16 ? launch_resident<1, BF>(p, s) : launch_resident<2, BF>(p, s);
  if constexpr (!BF)
    if (p.M > 16) return launch_stream<2, false>(p, s);
  return launch_stream<1, BF>(p, s);
}

int launch_many(Fp8Params& p, hipStream_t s) {
  // Large tiles read their operands less often, small ones leave fewer compute units idle: the fewest rounds, a round of 256 x 256
  // (256 at a time) counted as 20, of 256 x 128 as 13, of 128 x 64 (512 at a time) as 10.  (us in the three, K = 3584: 600 rows
  // x 18944 49, 59, 64; 300 rows 44, 31, 42; 129 rows 39, 27, 22; 100 rows x 37888 42, 29, 37; 300 rows x 37888 84, 58, 74)
  const auto tiles = [&](long tm, long tn) { return ((p.N + tm - 1) / tm) * ((p.M + tn - 1) / tn); };
  const long l = 20 * ((tiles(256, 256) + 255) / 256), m = 13 * ((tiles(256, 128) + 255) / 256), t = 10 * ((tiles(128, 64) + 511) / 512);
  if (l <= m && l <= t) return launch_fp8<TileL>(p, s);
  if (m <= t) return launch_fp8<TileM>(p, s);
  // Few tiles of a long k wait for one stage after the other, 0.4 us each behind a start and end of 3 us; the streaming kernel, 32
  // rows at a time, has all of k on its way at once, but reads rows and features once per workgroup, at 9 TB/s out of L2.
  // (us by tiles and streamed: 59 rows x 280 x 8304 28.8 and 10.2, 64 x 4096 x 4096 16.2 and 13.6, 333 x 2201 x 1168 10.7 and 7.7;
  // 1398 x 304 x 4688 18.8 and 21.6, 155 x 7585 x 8176 38 and 61)
  const long f = stream_wide(p) ? 32 : 16;
  const double read = (double)((p.M + 31) / 32 * ((p.N + f - 1) / f)) * (32 + f) * p.K;
  if (read < 9e6 * (3 + 0.4 * ((p.K + 127) / 128))) return launch_stream<2, false>(p, s);
  return launch_fp8<TileS2>(p, s);
}

constexpr int kFewRows = 32;
// bf16 rows streamed as they are (32 rows x 2048 x 8192: 20.6 us so, 16.0 with a launch that quantises them first)
constexpr int kFewBf16Rows = 16;

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
  const int groups = (k + 2047) / 2048;
  if (!launch_fits(n_rows * groups, 256)) return PDLLM_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(fp8_quantize_rows_kernel, dim3((unsigned)(n_rows * groups)), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const char*>(x), 2L * x_stride, groups, k,
                     static_cast<char*>(q), (long)q_stride, scale, (long)scale_row_stride, (long)scale_block_stride);
  return launch_status();
}

extern "C" int pdllm_fp8_quantize_blocks(const void* w, int64_t w_stride, int64_t n_rows, int32_t k, void* q, int64_t q_stride,
                                         float* scale, int64_t scale_row_stride, int64_t scale_block_stride,
                                         pdllm_stream_t stream) {
  const int st = check_quantize(w, w_stride, n_rows, k, q, q_stride, scale, scale_row_stride, scale_block_stride);
  if (st != PDLLM_OK || n_rows == 0) return st;
  const long blocks = (n_rows + 127) / 128 * ((k + 127) / 128);
  if (!launch_fits(blocks, 256)) return PDLLM_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(fp8_quantize_blocks_kernel, dim3((unsigned)blocks), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const char*>(w), 2L * w_stride, (long)n_rows, k, static_cast<char*>(q), (long)q_stride, scale,
                     (long)scale_row_stride, (long)scale_block_stride);
  return launch_status();
}

namespace pdllm {
namespace {

int check_linear(int64_t m, int64_t n, int32_t k) {
  return m < 0 || n <= 0 || k <= 0 || k % 16 || k > (1 << 20) || m > kMaxRows || n > (1L << 30) ? PDLLM_ERR_SHAPE : PDLLM_OK;
}
// operands of elem bytes per value of x
int check_linear_strides(const void* x, int64_t x_stride, int elem, const void* weight, int64_t weight_stride, int64_t sw_row,
                         int64_t sw_blk, int64_t n, int32_t k, const void* out, int64_t out_stride) {
  if (x_stride < k || (elem * x_stride) % 16 || weight_stride < k || weight_stride % 16 || (uintptr_t)x % 16 ||
      (uintptr_t)weight % 16 || elem * x_stride * 256 >= 0x7fffffffL || weight_stride * 256 >= 0x7fffffffL || out_stride < n ||
      sw_row < 0 || sw_blk < 0 || (uintptr_t)out % 2)
    return PDLLM_ERR_STRIDE;
  return PDLLM_OK;
}
Fp8Params linear_params(const void* x, int64_t x_bytes, const void* weight, int64_t weight_stride, const float* weight_scale,
                        int64_t sw_row, int64_t sw_blk, int64_t m, int64_t n, int32_t k, void* out, int64_t out_stride) {
  Fp8Params p = {};
  p.x = static_cast<const char*>(x);
  p.w = static_cast<const char*>(weight);
  p.sw = weight_scale;
  p.x_stride = x_bytes;
  p.w_stride = weight_stride;
  p.sw_row = sw_row;
  p.sw_blk = sw_blk;
  p.M = m;
  p.N = n;
  p.K = k;
  p.out = static_cast<__bf16*>(out);
  p.o_stride = out_stride;
  return p;
}

}  // namespace
}  // namespace pdllm

extern "C" int pdllm_fp8_linear(const void* x, int64_t x_stride, const float* x_scale, int64_t x_scale_row_stride,
                                int64_t x_scale_block_stride, const void* weight, int64_t weight_stride,
                                const float* weight_scale, int64_t weight_scale_row_stride,
                                int64_t weight_scale_block_stride, int64_t m, int64_t n, int32_t k, void* out,
                                int64_t out_stride, pdllm_stream_t stream) {
  int st = check_linear(m, n, k);
  if (st != PDLLM_OK || m == 0) return st;
  if (!x || !x_scale || !weight || !weight_scale || !out) return PDLLM_ERR_NULL;
  st = check_linear_strides(x, x_stride, 1, weight, weight_stride, weight_scale_row_stride, weight_scale_block_stride, n, k, out,
                            out_stride);
  if (st != PDLLM_OK) return st;
  if (x_scale_row_stride < 0 || x_scale_row_stride >= (1 << 22) || x_scale_block_stride < 0) return PDLLM_ERR_STRIDE;
  Fp8Params p = linear_params(x, x_stride, weight, weight_stride, weight_scale, weight_scale_row_stride,
                              weight_scale_block_stride, m, n, k, out, out_stride);
  p.sx = x_scale;
  p.sx_row = x_scale_row_stride;
  p.sx_blk = x_scale_block_stride;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return m <= kFewRows ? launch_few<false>(p, s) : launch_many(p, s);
}

extern "C" int64_t pdllm_fp8_linear_bf16_workspace_bytes(int64_t m, int32_t k) {
  if (check_linear(m, 1, k) != PDLLM_OK) return PDLLM_ERR_SHAPE;
  return m <= kFewBf16Rows ? 0 : m * k + 4 * m * ((k + 127) / 128);
}

extern "C" int pdllm_fp8_linear_bf16(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
                                     const float* weight_scale, int64_t weight_scale_row_stride,
                                     int64_t weight_scale_block_stride, int64_t m, int64_t n, int32_t k, void* workspace,
                                     int64_t workspace_bytes, void* out, int64_t out_stride, pdllm_stream_t stream) {
  int st = check_linear(m, n, k);
  if (st != PDLLM_OK || m == 0) return st;
  if (!x || !weight || !weight_scale || !out) return PDLLM_ERR_NULL;
  st = check_linear_strides(x, x_stride, 2, weight, weight_stride, weight_scale_row_stride, weight_scale_block_stride, n, k, out,
                            out_stride);
  if (st != PDLLM_OK) return st;
  Fp8Params p = linear_params(x, 2 * x_stride, weight, weight_stride, weight_scale, weight_scale_row_stride,
                              weight_scale_block_stride, m, n, k, out, out_stride);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (m > kFewBf16Rows && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < pdllm_fp8_linear_bf16_workspace_bytes(m, k)))
    return PDLLM_ERR_WORKSPACE;
  if (m <= kFewBf16Rows || resident_fits(p, true)) return launch_few<true>(p, s);  // quantised where they are read: one launch
  char* q = static_cast<char*>(workspace);
  float* scale = reinterpret_cast<float*>(q + m * k);
  st = pdllm_fp8_quantize_rows(x, x_stride, m, k, q, k, scale, 1, m, stream);
  if (st != PDLLM_OK) return st;
  p.x = q;
  p.x_stride = k;
  p.sx = scale;
  p.sx_row = 1;
  p.sx_blk = m;
  return m <= kFewRows ? launch_few<false>(p, s) : launch_many(p, s);
}
