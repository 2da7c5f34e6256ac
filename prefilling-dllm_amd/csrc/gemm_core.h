// The matrix-product loop shared by the vocabulary-head and fp8 kernels for gfx950: one workgroup forms a tile
// C[m][n] = sum_k A[m][k] B[n][k] on the matrix cores, fp32 accumulation.
//
// Orientation.  A is the operand whose index is contiguous in the output (vocabulary entries, output features, state
// columns), B the one over rows (tokens): in the result layouts of the matrix instructions a lane then owns ONE row of the output
// and groups of four neighbouring columns, so softmax statistics of a row are sums over a lane's own registers.
//
// LDS.  A stage holds KB = 128 bytes of k (a cache line) per row of A and of B.  Operands that lie with k contiguous ("KC") are
// kept as rows of 128 bytes, 16-byte chunk c of row r at position c ^ ((r >> 1) & 7): 16 consecutive rows of one chunk cover all 64
// banks.  Operands that lie with k as their row index ("KS", bf16 only) are kept as 64 rows of TM * 2 bytes, chunk c of row
// r at c ^ ks_xor(r), and read through the transposing 64-bit reads (half a wave takes four rows and the four 8 rows further on,
// two neighbouring chunks of each: again all banks).  Copies go straight from memory to LDS, up to ST stages ahead; operand
// reads are hand-issued with counted waits so that they do not wait for the copies.
#pragma once

#include <type_traits>
#include <utility>

#include "attn_common.h"

namespace pdllm {

template <int N>
__device__ __forceinline__ void vm_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ void lgkm_wait() {
  asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wg_barrier() {
  asm volatile("s_barrier" ::: "memory");
}

// position of a row's chunks in LDS (see above)
constexpr int KB = 128;  // bytes of k in a stage
__device__ __forceinline__ constexpr unsigned kc_xor(unsigned row) { return (row >> 1) & 7; }
__device__ __forceinline__ constexpr unsigned ks_xor(unsigned row) { return (row & 3) << 2 | ((row >> 2) & 2); }

typedef __attribute__((address_space(3))) void lds_void;
__device__ __forceinline__ lds_void* lds_at(unsigned a) { return (lds_void*)(size_t)a; }

constexpr unsigned kOutOfRange = 0x80000000u;  // an offset behind every buffer (their sizes stay below 2 GiB)

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, unsigned bytes) {
  // the same in every lane; said explicitly, since 64-bit comparisons on the way leave the scalar registers
  const uint64_t a = (uint64_t)base;
  const uint64_t lo = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)a);
  const uint64_t hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc((void*)(hi << 32 | lo), 0, __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}

// Rows of k-contiguous data, through a buffer whose size ends with the last valid row: rows and k behind the end read
// as zero.  L copies of 8 rows per wave and stage; a lane's offset inside them takes one of two values (the chunk positions of even
// and odd groups of 8 rows), the group goes through the buffer's base.
template <int L>
struct LoadKC {
  static constexpr int R = 1024 / KB, LANES = KB / 16;  // rows of a copy, lanes of a row
  const char* base;  // first row of the wave
  int bytes;         // from there to the end of the last valid row; not positive: none
  unsigned stride, kbytes, off[2], kc[2];
  __device__ __forceinline__ void init(const void* b, long rows_left, unsigned row_bytes, unsigned kb, int wave, int lane) {
    base = static_cast<const char*>(b) + (long)(R * wave * L) * row_bytes;
    rows_left -= R * wave * L;
    const int rows = rows_left < 0 ? 0 : (rows_left < R * L ? (int)rows_left : R * L);
    bytes = rows > 0 ? (int)((rows - 1) * row_bytes + kb) : 0;
    stride = row_bytes;
    kbytes = kb;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const unsigned c = (lane % LANES) ^ kc_xor(R * (wave * L + q) + lane / LANES);
      kc[q] = 16 * c;
      off[q] = (lane / LANES) * row_bytes + 16 * c;
    }
  }
  template <int I>
  __device__ __forceinline__ void one(int t, unsigned dst) const {
    const unsigned k = (unsigned)KB * t;
    const unsigned o = k + kc[I & 1] < kbytes ? off[I & 1] + k : kOutOfRange;
    const int left = bytes - (int)(R * I * stride);
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(base + (long)(R * I) * stride, left > 0 ? left : 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, lds_at(dst + 1024 * I), 16, o, 0, 0, 0);
  }
};

// Rows of k-contiguous data at a 64-bit address per row (rows gathered from two tensors).  Rows past the end repeat a
// valid row (their results are dropped); k behind the end repeats the row's first bytes (the other operand is zero
// there).
template <int L>
struct LoadRows {
  static constexpr int R = 1024 / KB, LANES = KB / 16;
  const char* p[L];
  unsigned kc[2], kbytes;
  template <typename F>
  __device__ __forceinline__ void init(F&& row_ptr, unsigned kb, int wave, int lane) {
    kbytes = kb;
#pragma unroll
    for (int i = 0; i < L; ++i) p[i] = row_ptr((unsigned)(R * (wave * L + i) + lane / LANES));
#pragma unroll
    for (int q = 0; q < 2; ++q) kc[q] = 16 * ((lane % LANES) ^ kc_xor(R * (wave * L + q) + lane / LANES));
  }
  template <int I>
  __device__ __forceinline__ void one(int t, unsigned dst) const {
    const unsigned k = (unsigned)KB * t;
    const unsigned o = k + kc[I & 1] < kbytes ? k + kc[I & 1] : 0u;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(p[I] + o), lds_at(dst + 1024 * I), 16, 0, 0);
  }
};

// KB / 2 rows of k per stage, W columns (bf16) of each: base = first row, first column.  Rows from k_rows on read as zero;
// so do columns from col_bytes on.
template <int L, int W>
struct LoadKS {
  static constexpr int ROWS = KB / 2, CH = W / 8;  // rows of a stage, chunks of a row
  const char* base;
  long stride;  // bytes
  long k_rows;
  unsigned off[L], colb;
  __device__ __forceinline__ void init(const void* b, long stride_bytes, long rows, unsigned col_bytes, int wave, int lane) {
    base = static_cast<const char*>(b);
    stride = stride_bytes;
    k_rows = rows;
    colb = col_bytes;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const unsigned q = 64 * (wave * L + i) + lane;
      const unsigned row = q / CH, c = (q % CH) ^ ks_xor(row);
      off[i] = 16 * c < col_bytes ? row * (unsigned)stride_bytes + 16 * c : kOutOfRange;
    }
  }
  template <int I>
  __device__ __forceinline__ void one(int t, unsigned dst) const {
    const long r0 = (long)ROWS * t;
    const long left = k_rows - r0;
    const unsigned rows = left <= 0 ? 0u : (left < ROWS ? (unsigned)left : (unsigned)ROWS);
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(base + r0 * stride, rows ? (rows - 1) * (unsigned)stride + colb : 0u);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, lds_at(dst + 1024 * I), 16, off[I], 0, 0, 0);
  }
};

template <int MT_, int NT_, int WM_, int WN_, int ST_>
struct Tile {
  static constexpr int MT = MT_, NT = NT_, WM = WM_, WN = WN_, ST = ST_;
  static constexpr int NW = WM * WN, THREADS = 64 * NW;
  static constexpr int TM = 32 * MT * WM, TN = 32 * NT * WN;
  static constexpr int A_BYTES = TM * KB, B_BYTES = TN * KB, STAGE = A_BYTES + B_BYTES;
  static constexpr int LA = A_BYTES / 1024 / NW, LB = B_BYTES / 1024 / NW;
  static_assert(LA * NW * 1024 == A_BYTES && LB * NW * 1024 == B_BYTES, "every wave copies the same number of pieces");
  static constexpr int LDS = ST * STAGE;
  static_assert(LDS <= 160 * 1024, "LDS of a compute unit");
};

template <class F, int... I>
__device__ __forceinline__ void unroll_over(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
// f(0), f(1), ... f(N - 1), each with its number as a constant
template <int N, class F>
__device__ __forceinline__ void unrolled(F&& f) {
  unroll_over(f, std::make_integer_sequence<int, N>{});
}

// A wave's bf16 operand fragments for the 16x16x32 instruction: blocks of 16 rows (KC) or columns (KS), the first one at `first` of
// the tile.  A fragment of step ks holds, in lanes 16 g .. 16 g + 15, the k values 32 ks + 8 g .. + 7 of its 16 rows.
template <bool KS, int W>
struct Frag;
template <int W>
struct Frag<false, W> {
  unsigned a[2];
  typedef bf16x8 raw;
  static constexpr int READS = 1;  // LDS operations per fragment
  __device__ __forceinline__ void init(unsigned lds_base, int first, int lane) {
    const int l16 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) a[ks] = lds_base + (first + l16) * KB + (((4 * ks + g) ^ kc_xor(l16)) << 4);
  }
  template <int KS_, int J>
  __device__ __forceinline__ void read(raw& d, unsigned stage) const {
    lds_read_b128<J * 16 * KB>(d, a[KS_] + stage);
  }
  static __device__ __forceinline__ bf16x8 value(const raw& r) { return r; }
};
struct TrPair {
  s16x4 lo, hi;
};
template <int W>
struct Frag<true, W> {
  static_assert(W >= 128, "the chunks of a row change places in groups of 16");
  unsigned a;
  typedef TrPair raw;
  static constexpr int READS = 2;
  __device__ __forceinline__ void init(unsigned lds_base, int first, int lane) {
    const int l16 = lane & 15, g = lane >> 4;
    const int row = 8 * g + (l16 >> 2);
    a = lds_base + row * (W * 2) + ((((unsigned)first / 8 + ((l16 & 3) >> 1)) ^ ks_xor(row)) << 4) + ((l16 & 1) << 3);
  }
  // (`first` is a multiple of the wave's columns, a power of two: block J is two chunks further, by an exclusive or)
  template <int KS_, int J>
  __device__ __forceinline__ void read(raw& d, unsigned stage) const {
    lds_read_tr16_b64<32 * KS_ * W * 2>(d.lo, (a ^ (32 * J)) + stage);
    lds_read_tr16_b64<(32 * KS_ + 4) * W * 2>(d.hi, (a ^ (32 * J)) + stage);
  }
  static __device__ __forceinline__ bf16x8 value(const raw& r) {
    typedef __attribute__((ext_vector_type(8))) short s16x8;
    const s16x8 v = __builtin_shufflevector(r.lo, r.hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, v);
  }
};
// Ties a wait that has been issued to the registers the reads before it filled: nothing that uses them moves above it.
__device__ __forceinline__ void tie(bf16x8& r) { asm volatile("" : "+v"(r)::"memory"); }
__device__ __forceinline__ void tie(TrPair& r) { asm volatile("" : "+v"(r.lo), "+v"(r.hi)::"memory"); }

// A wave's bf16 accumulators: blocks of 16 x 16, lane 16 g + l holds entries 4 g .. 4 g + 3 of A's block and row l of B's.
template <class T>
struct Acc {
  f32x4 v[2 * T::MT][2 * T::NT];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 2 * T::MT; ++i)
#pragma unroll
      for (int j = 0; j < 2 * T::NT; ++j) v[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
};

// The bf16 loop over `steps` stages.  issue(t, lds address of the stage, i) starts copy i of this wave's T::LA + T::LB of stage t.
// A stage is two steps of k = 32 in four turns, half of the wave's blocks of A each; the fragments of the next turn are read
// while a turn's matrix instructions run.  One barrier per stage, in front of the last turn: by then every wave has read all of
// the stage and its own part of the next one has landed, so behind the barrier the stage's buffer takes the copies of
// stage t + ST, half of them in this turn and half in the next.
// The 16x16x32 instruction, not 32x32x16: the large products here run at the card's power limit, and with operands of normally
// distributed values out of registers the one sustains 2050 TFLOP/s, the other 1340 to 1640 (zeros: 2450 and 1810 to 2210).
// 4096 rows x 152064 x 3584, scores only: 3.69 ms with 32x32x16, 3.47 ms so; 3.29 ms with the instructions of a turn in a fixed
// order in which neighbours share an operand; 3.16 ms with reads and copies between them and no branch in the loop (3.14 to 3.21 ms since
// the statistics behind it are taken in groups of 64 entries).
template <class T, bool AKS, bool BKS, class Issue>
__device__ __forceinline__ void mainloop_bf16(Acc<T>& acc, int steps, unsigned lds_base, Issue&& issue) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / T::WN, wn = wave % T::WN;
  constexpr int COPIES = T::LA + T::LB, MT = T::MT, NT = T::NT;
  typedef Frag<AKS, T::TM> FA;
  typedef Frag<BKS, T::TN> FB;
  FA fa;
  FB fb;
  fa.init(lds_base, wm * MT * 32, lane);
  fb.init(lds_base + T::A_BYTES, wn * NT * 32, lane);
  typename FA::raw A[2][MT];      // of this turn and the next
  typename FB::raw B[2][2 * NT];  // of both steps
  constexpr int RA = MT * FA::READS, RB = NT * FB::READS;
  static_assert(RA + RB <= 15, "the wait counts 15 LDS operations at most");
  acc.clear();
  if (steps <= 0) return;
  // fragment n of those that a turn reads for the next: blocks of A, then of B
  auto read_a = [&](auto turn, auto n, unsigned cur) __attribute__((always_inline)) {
    constexpr int U = decltype(turn)::value, i = decltype(n)::value;
    fa.template read<U / 2, (U & 1) * MT + i>(A[U & 1][i], cur);
  };
  auto read_b = [&](auto ks, auto n, unsigned cur) __attribute__((always_inline)) {
    constexpr int S = decltype(ks)::value, j = decltype(n)::value;
    fb.template read<S, j>(B[S][j], cur);
  };
  // the matrix instructions of a turn in a fixed order, neighbours sharing an operand; behind instruction n: between(n)
  constexpr int PRODUCTS = MT * 2 * NT;
  auto mul = [&](auto turn, auto&& between) __attribute__((always_inline)) {
    constexpr int U = decltype(turn)::value, S = U / 2, H = U & 1;
#pragma unroll
    for (int i = 0; i < MT; ++i) tie(A[H][i]);
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) tie(B[S][j]);
    unrolled<PRODUCTS>([&](auto n) __attribute__((always_inline)) {
      constexpr int i = decltype(n)::value / (2 * NT), q = decltype(n)::value % (2 * NT), j = i % 2 ? 2 * NT - 1 - q : q;
      acc.v[H * MT + i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(FA::value(A[H][i]), FB::value(B[S][j]), acc.v[H * MT + i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      between(n);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  constexpr std::integral_constant<int, 0> c0{};
  constexpr std::integral_constant<int, 1> c1{};
  constexpr std::integral_constant<int, 2> c2{};
  constexpr std::integral_constant<int, 3> c3{};
  constexpr int HALF = COPIES / 2;
  // Turns of many instructions have their reads and copies between them, and the loop no branches: copies of stages behind the
  // last one read nothing, or the first bytes of a row.  Short turns (tiles of few rows, which wait for memory) read first.
  constexpr bool SPREAD = PRODUCTS >= 16;
  auto copy = [&](int s, unsigned at, auto k) __attribute__((always_inline)) {
    if (SPREAD || s < steps) issue(s, lds_base + at, k);
  };
  // a turn: its matrix instructions, the reads of the next one and copies
  auto turn = [&](auto u, auto reads, auto&& read, auto copies, auto&& next) __attribute__((always_inline)) {
    constexpr int R = decltype(reads)::value, C = decltype(copies)::value;
    if constexpr (SPREAD) {
      lgkm_wait<0>();
      mul(u, [&](auto n) __attribute__((always_inline)) {
        constexpr int at = decltype(n)::value;
        unrolled<R>([&](auto k) __attribute__((always_inline)) { if constexpr (decltype(k)::value * PRODUCTS / (R + 6) == at) read(k); });
        unrolled<C>([&](auto k) __attribute__((always_inline)) { if constexpr (((2 * decltype(k)::value + 1) * PRODUCTS) / (2 * C) == at) next(k); });
      });
    } else {
      constexpr int OPS = decltype(u)::value == 3 ? 0 : decltype(u)::value == 2 ? RA : RA + RB;
      unrolled<R>(read);
      if constexpr (decltype(u)::value != 3) lgkm_wait<OPS>();
      unrolled<C>(next);
      mul(u, [](auto) {});
    }
  };
  // (the second half of stage ST - 1 is copied in the first turn)
  unrolled<T::ST * COPIES - (COPIES - HALF)>([&](auto n) __attribute__((always_inline)) {
    constexpr int s = decltype(n)::value / COPIES;
    copy(s, s * T::STAGE, std::integral_constant<int, decltype(n)::value % COPIES>{});
  });
  unsigned cur = 0, old = (T::ST - 1) * T::STAGE;
  if (SPREAD || steps >= T::ST) vm_wait<(T::ST - 2) * COPIES + HALF>();
  else vm_wait<0>();
  wg_barrier();
  unrolled<2 * NT>([&](auto j) __attribute__((always_inline)) { read_b(c0, j, cur); });
  unrolled<MT>([&](auto i) __attribute__((always_inline)) { read_a(c0, i, cur); });
  typedef std::integral_constant<int, MT + NT> ReadsAB;
  auto none = [](auto) {};
  int t = 0;
  do {
    turn(c0, ReadsAB{}, [&](auto k) __attribute__((always_inline)) {
          constexpr int n = decltype(k)::value;
          if constexpr (n < MT) read_a(c1, k, cur);
          else read_b(c1, std::integral_constant<int, n - MT>{}, cur);
        }, std::integral_constant<int, COPIES - HALF>{}, [&](auto k) __attribute__((always_inline)) {
          copy(t + T::ST - 1, old, std::integral_constant<int, HALF + decltype(k)::value>{});
        });
    turn(c1, ReadsAB{}, [&](auto k) __attribute__((always_inline)) {
          constexpr int n = decltype(k)::value;
          if constexpr (n < MT) read_a(c2, k, cur);
          else read_b(c1, std::integral_constant<int, NT + n - MT>{}, cur);
        }, c0, none);
    turn(c2, std::integral_constant<int, MT>{}, [&](auto k) __attribute__((always_inline)) { read_a(c3, k, cur); }, c0, none);
    lgkm_wait<0>();
    if (SPREAD || t + T::ST - 1 < steps) vm_wait<(T::ST - 2) * COPIES>();
    else vm_wait<0>();
    wg_barrier();
    old = cur;
    cur = cur == (T::ST - 1) * T::STAGE ? 0u : cur + T::STAGE;
    // (behind the last stage: reads of whatever the buffer holds, which nothing uses)
    turn(c3, std::integral_constant<int, MT + 2 * NT>{}, [&](auto k) __attribute__((always_inline)) {
          constexpr int n = decltype(k)::value;
          if constexpr (n < 2 * NT) read_b(c0, k, cur);
          else read_a(c0, std::integral_constant<int, n - 2 * NT>{}, cur);
        }, std::integral_constant<int, HALF>{}, [&](auto k) __attribute__((always_inline)) { copy(t + T::ST, old, k); });
  } while (++t < steps);
  lgkm_wait<0>();
#pragma unroll
  for (int i = 0; i < MT; ++i) tie(A[0][i]);
#pragma unroll
  for (int j = 0; j < 2 * NT; ++j) tie(B[0][j]);
  vm_wait<0>();  // (the caller's barrier follows before the buffers are used for something else)
}

// A bf16 tile to memory through LDS, so that rows leave in whole lines: 16 bytes a lane where the rows begin at multiples of
// that, else words.  fill(put) hands over the wave's results: put(row, column, four values) with columns in multiples of four.
template <class T, class Fill>
__device__ __forceinline__ void store_tile(char* lds, Fill&& fill, __bf16* out, long stride, long rows, long cols) {
  constexpr int CH = T::TM / 8;  // chunks of a row
  static_assert(T::TM * T::TN * 2 <= T::LDS && CH >= 16, "the results take the place of the operands");
  __syncthreads();  // the tile's operands are done with
  fill([&](int r, int c, uint2 v) __attribute__((always_inline)) {
    *reinterpret_cast<uint2*>(lds + (r * CH + ((c >> 3) ^ (r & 15))) * 16 + 2 * (c & 4)) = v;
  });
  __syncthreads();
  const int nr = rows < T::TN ? (int)rows : T::TN, nc = cols < T::TM ? (int)cols : T::TM;
  const unsigned odd = (unsigned)(uintptr_t)out | (unsigned)(2 * stride);
  if (odd % 16 == 0) {
    for (int k = threadIdx.x; k < nr * CH; k += T::THREADS) {
      const int r = k / CH, c = k % CH;
      const uint4 v = *reinterpret_cast<const uint4*>(lds + (r * CH + (c ^ (r & 15))) * 16);
      __bf16* o = out + r * stride + 8 * c;
      if (8 * c + 8 <= nc) {
        *reinterpret_cast<uint4*>(o) = v;
      } else {
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (8 * c + e < nc) reinterpret_cast<unsigned short*>(o)[e] = (unsigned short)(w[e >> 1] >> (16 * (e & 1)));
      }
    }
  } else if (odd % 4 == 0) {
    for (int k = threadIdx.x; k < nr * (T::TM / 2); k += T::THREADS) {
      const int r = k / (T::TM / 2), c = k % (T::TM / 2);
      const unsigned v = *reinterpret_cast<const unsigned*>(lds + (r * CH + ((c >> 2) ^ (r & 15))) * 16 + 4 * (c & 3));
      __bf16* o = out + r * stride + 2 * c;
      if (2 * c + 2 <= nc) *reinterpret_cast<unsigned*>(o) = v;
      else if (2 * c < nc) *reinterpret_cast<unsigned short*>(o) = (unsigned short)v;
    }
  } else {
    // rows that begin between two words: word k of a row holds its elements 2 k - p and 2 k - p + 1, p = the row's parity
    constexpr int WORDS = T::TM / 2 + 1;
#pragma unroll 4
    for (int i = threadIdx.x; i < nr * WORDS; i += T::THREADS) {
      const int r = i / WORDS, k = i % WORDS;
      unsigned short* o = reinterpret_cast<unsigned short*>(out + r * stride);
      const int c = 2 * k - ((int)((uintptr_t)o >> 1) & 1);
      auto at = [&](int e) __attribute__((always_inline)) {
        return *reinterpret_cast<const unsigned short*>(lds + (r * CH + ((e >> 3) ^ (r & 15))) * 16 + 2 * (e & 7));
      };
      const unsigned lo = c >= 0 ? at(c) : 0u, hi = c + 1 < T::TM ? at(c + 1) : 0u;
      if (c >= 0 && c + 1 < nc) *reinterpret_cast<unsigned*>(o + c) = lo | hi << 16;
      else if (c >= 0 && c < nc) o[c] = (unsigned short)lo;
      else if (c < 0) o[0] = (unsigned short)hi;
    }
  }
}

// The wave's accumulators, packed in pairs, by store_tile.
template <class T, class Pack>
__device__ __forceinline__ void store_acc(char* lds, const Acc<T>& acc, Pack&& pack, __bf16* out, long stride, long rows, long cols) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r0 = wave % T::WN * (32 * T::NT) + (lane & 15), c0 = wave / T::WN * (32 * T::MT) + 4 * (lane >> 4);
  store_tile<T>(
      lds,
      [&](auto&& put) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2 * T::NT; ++j)
#pragma unroll
          for (int i = 0; i < 2 * T::MT; ++i)
            put(r0 + 16 * j, c0 + 16 * i, make_uint2(pack(acc.v[i][j][0], acc.v[i][j][1]), pack(acc.v[i][j][2], acc.v[i][j][3])));
      },
      out, stride, rows, cols);
}

}  // namespace pdllm
