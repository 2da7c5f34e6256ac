// The matrix-product loop shared by the vocabulary-head and fp8 kernels for gfx950: one workgroup forms a tile
// C[m][n] = sum_k A[m][k] B[n][k] on the matrix cores, fp32 accumulation.
//
// Orientation.  A is the operand whose index is contiguous in the output (vocabulary entries, output features, state
// columns), B the one over rows (tokens): in the 32x32 result layout a lane then owns ONE row of the output (lane & 31)
// and 16 of its columns in registers, so softmax statistics of a row are sums over a lane's own registers and
// stores are groups of four neighbouring columns.
//
// LDS.  A stage holds KB = 64 or 128 bytes of k per row of A and of B.  Operands that lie with k contiguous ("KC") are kept as
// rows of KB bytes, 16-byte chunk c of row r at position c ^ x(r) with x(r) = (r >> 1) & 7 (KB = 128) or (r >> 2) & 3 (KB = 64):
// 16 consecutive rows of one chunk cover all 64 banks.  Operands that lie with k as their row index ("KS", bf16 only) are kept
// as KB / 2 rows of TM * 2 bytes, chunk c of row r at c ^ ((r & 3) << 2), and read through the transposing 64-bit reads
// (four rows of four neighbouring chunks per half wave, again all banks).  Copies go straight from memory to LDS, up to ST
// stages ahead; operand reads are hand-issued with counted waits so that they do not wait for the copies.
//
// KB = 128 reads whole cache lines of a row at a time and is what the tiles of few rows use, which wait for memory; KB = 64
// gives the large tiles four stages in 128 KB, so that the copies can be issued two at a time between groups of matrix
// instructions instead of eight in a row, which kept the matrix unit waiting behind the address unit.
#pragma once

#include <type_traits>

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
template <int KB>
__device__ __forceinline__ constexpr unsigned chunk_xor(unsigned row) {
  return KB == 128 ? (row >> 1) & 7 : (row >> 2) & 3;
}

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
// as zero.  L copies of 1024 / KB rows per wave and stage; a lane's offset inside them takes one of two values (KB = 128: the
// chunk positions of even and odd groups of 8 rows), the group goes through the buffer's base.
template <int L, int KB = 128>
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
      const unsigned c = (lane % LANES) ^ chunk_xor<KB>(R * (wave * L + q) + lane / LANES);
      kc[q] = 16 * c;
      off[q] = (lane / LANES) * row_bytes + 16 * c;
    }
  }
  __device__ __forceinline__ void issue(int t, unsigned dst) const {
    const unsigned k = (unsigned)KB * t;
    unsigned o[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) o[q] = k + kc[q] < kbytes ? off[q] + k : kOutOfRange;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int left = bytes - (int)(R * i * stride);
      const __amdgpu_buffer_rsrc_t rs = make_rsrc(base + (long)(R * i) * stride, left > 0 ? left : 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, lds_at(dst + 1024 * i), 16, o[KB == 128 ? i & 1 : 0], 0, 0, 0);
    }
  }
};

// Rows of k-contiguous data at a 64-bit address per row (rows gathered from two tensors).  Rows past the end repeat a
// valid row (their results are dropped); k behind the end repeats the row's first bytes (the other operand is zero
// there).
template <int L, int KB = 128>
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
    for (int q = 0; q < 2; ++q) kc[q] = 16 * ((lane % LANES) ^ chunk_xor<KB>(R * (wave * L + q) + lane / LANES));
  }
  __device__ __forceinline__ void issue(int t, unsigned dst) const {
    const unsigned k = (unsigned)KB * t;
    unsigned o[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) o[q] = k + kc[q] < kbytes ? k + kc[q] : 0u;
#pragma unroll
    for (int i = 0; i < L; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(p[i] + o[KB == 128 ? i & 1 : 0]),
                                       lds_at(dst + 1024 * i), 16, 0, 0);
  }
};

// KB / 2 rows of k per stage, W columns (bf16) of each: base = first row, first column.  Rows from k_rows on read as zero;
// so do columns from col_bytes on.
template <int L, int W, int KB = 128>
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
      const unsigned row = q / CH, c = (q % CH) ^ ((row & 3) << 2);
      off[i] = 16 * c < col_bytes ? row * (unsigned)stride_bytes + 16 * c : kOutOfRange;
    }
  }
  __device__ __forceinline__ void issue(int t, unsigned dst) const {
    const long r0 = (long)ROWS * t;
    const long left = k_rows - r0;
    const unsigned rows = left <= 0 ? 0u : (left < ROWS ? (unsigned)left : (unsigned)ROWS);
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(base + r0 * stride, rows ? (rows - 1) * (unsigned)stride + colb : 0u);
#pragma unroll
    for (int i = 0; i < L; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, lds_at(dst + 1024 * i), 16, off[i], 0, 0, 0);
  }
};

template <int MT_, int NT_, int WM_, int WN_, int ST_, int KB_ = 128>
struct Tile {
  static constexpr int MT = MT_, NT = NT_, WM = WM_, WN = WN_, ST = ST_, KB = KB_;
  static constexpr int NW = WM * WN, THREADS = 64 * NW;
  static constexpr int TM = 32 * MT * WM, TN = 32 * NT * WN;
  static constexpr int A_BYTES = TM * KB, B_BYTES = TN * KB, STAGE = A_BYTES + B_BYTES;
  static constexpr int LA = A_BYTES / 1024 / NW, LB = B_BYTES / 1024 / NW;
  static_assert(LA * NW * 1024 == A_BYTES && LB * NW * 1024 == B_BYTES, "every wave copies the same number of pieces");
  static constexpr int LDS = ST * STAGE;
  static_assert(LDS <= 160 * 1024, "LDS of a compute unit");
};

// A wave's operand fragments: N_ blocks of 32 rows (KC) or columns (KS), the first one at `first` of the tile.  A fragment of
// step ks holds, in lane half h, the k values 16 ks + 8 h .. + 7 (bf16) of its row; for fp8 two fragments make one operand
// (the k values of both operands are permuted alike, which a sum over k does not see).
template <int N_, bool KS, int W, int KB>
struct Frag;
template <int N_, int W, int KB>
struct Frag<N_, false, W, KB> {
  unsigned a[KB / 32];
  typedef bf16x8 raw;
  static constexpr int READS = 1;  // LDS operations per fragment
  __device__ __forceinline__ void init(unsigned lds_base, int first, int lane) {
    const int l32 = lane & 31, h = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < KB / 32; ++ks) a[ks] = lds_base + (first + l32) * KB + (((2 * ks + h) ^ chunk_xor<KB>(l32)) << 4);
  }
  template <int KS_, int J>
  __device__ __forceinline__ void read(raw& d, unsigned stage) const {
    lds_read_b128<J * 32 * KB>(d, a[KS_] + stage);
  }
  static __device__ __forceinline__ bf16x8 value(const raw& r) { return r; }
};
struct TrPair {
  s16x4 lo, hi;
};
template <int N_, int W, int KB>
struct Frag<N_, true, W, KB> {
  unsigned a[N_];
  typedef TrPair raw;
  static constexpr int READS = 2;
  __device__ __forceinline__ void init(unsigned lds_base, int first, int lane) {
    const int l32 = lane & 31, h = lane >> 5, i16 = lane & 15, g = l32 >> 4;
    const int row = 8 * h + (i16 >> 2);
#pragma unroll
    for (int j = 0; j < N_; ++j) {
      const int c = (first + 32 * j) / 8 + 2 * g + ((i16 & 3) >> 1);
      a[j] = lds_base + row * (W * 2) + ((c ^ ((row & 3) << 2)) << 4) + ((i16 & 1) << 3);
    }
  }
  template <int KS_, int J>
  __device__ __forceinline__ void read(raw& d, unsigned stage) const {
    lds_read_tr16_b64<(16 * KS_) * W * 2>(d.lo, a[J] + stage);
    lds_read_tr16_b64<(16 * KS_ + 4) * W * 2>(d.hi, a[J] + stage);
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

// The bf16 loop over `steps` stages.  issue(t, lds address of the stage, part) starts half of the copies of stage t (part 0
// or 1; T::LA + T::LB per wave in all).  One barrier per stage, in front of the stage's last group of matrix instructions: by
// then every wave has read all of the stage and its own part of the next one has landed, so behind the barrier the
// stage's buffer takes the copies of stage t + ST, half of them at once and half behind the next group, and the first
// fragments of the next stage are read while the last group runs.
template <class T, bool AKS, bool BKS, class Issue>
__device__ __forceinline__ void mainloop_bf16(f32x16 (&acc)[T::MT][T::NT], int steps, unsigned lds_base, Issue&& issue) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / T::WN, wn = wave % T::WN;
  constexpr int COPIES = T::LA + T::LB, GROUPS = T::KB / 32;
  typedef Frag<T::MT, AKS, T::TM, T::KB> FA;
  typedef Frag<T::NT, BKS, T::TN, T::KB> FB;
  FA fa;
  FB fb;
  fa.init(lds_base, wm * T::MT * 32, lane);
  fb.init(lds_base + T::A_BYTES, wn * T::NT * 32, lane);
  typename FA::raw A[2][T::MT];
  typename FB::raw B[2][T::NT];
  constexpr int READS = T::MT * FA::READS + T::NT * FB::READS;
  static_assert(READS <= 15, "the wait counts 15 LDS operations at most");
  static_assert(GROUPS == 2 || GROUPS == 4, "fragments alternate between two sets");
  if (steps <= 0) return;
  unsigned cur = 0, old = 0;
  auto read = [&](auto ks_tag, int set) __attribute__((always_inline)) {
    constexpr int KS = decltype(ks_tag)::value;
    fb.template read<KS, 0>(B[set][0], cur);
    if constexpr (T::NT > 1) fb.template read<KS, 1>(B[set][1], cur);
    fa.template read<KS, 0>(A[set][0], cur);
    if constexpr (T::MT > 1) fa.template read<KS, 1>(A[set][1], cur);
    if constexpr (T::MT > 2) fa.template read<KS, 2>(A[set][2], cur);
    if constexpr (T::MT > 3) fa.template read<KS, 3>(A[set][3], cur);
  };
  auto mul = [&](int set) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < T::MT; ++i) tie(A[set][i]);
#pragma unroll
    for (int j = 0; j < T::NT; ++j) tie(B[set][j]);
#pragma unroll
    for (int i = 0; i < T::MT; ++i)
#pragma unroll
      for (int j = 0; j < T::NT; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(FA::value(A[set][i]), FB::value(B[set][j]), acc[i][j], 0, 0, 0);
  };
#pragma unroll
  for (int s = 0; s < T::ST; ++s)
    if (s < steps) {
      issue(s, lds_base + s * T::STAGE, 0);
      issue(s, lds_base + s * T::STAGE, 1);
    }
  if (steps >= T::ST) vm_wait<(T::ST - 1) * COPIES>();
  else vm_wait<0>();
  wg_barrier();
  read(std::integral_constant<int, 0>{}, 0);
  // all groups of a stage but the last; behind the first one the second half of the copies that the barrier before allowed
  auto groups = [&](int t) __attribute__((always_inline)) {
    read(std::integral_constant<int, 1>{}, 1);
    lgkm_wait<READS>();
    if (t > 0 && t + T::ST - 1 < steps) issue(t + T::ST - 1, lds_base + old, 1);
    mul(0);
    if constexpr (GROUPS == 4) {
      read(std::integral_constant<int, 2>{}, 0);
      lgkm_wait<READS>();
      mul(1);
      read(std::integral_constant<int, 3>{}, 1);
      lgkm_wait<READS>();
      mul(0);
    }
    lgkm_wait<0>();
  };
  for (int t = 0; t < steps - 1; ++t) {
    groups(t);
    if (T::ST > 2 && t + T::ST - 1 < steps) vm_wait<(T::ST - 2) * COPIES>();
    else vm_wait<0>();
    wg_barrier();
    old = cur;
    cur = cur == (T::ST - 1) * T::STAGE ? 0u : cur + T::STAGE;
    read(std::integral_constant<int, 0>{}, 0);
    if (t + T::ST < steps) issue(t + T::ST, lds_base + old, 0);
    mul(1);
  }
  groups(steps - 1);
  mul(1);
}

// A tile of bf16 results to memory through LDS, so that a row's columns leave in one piece (a lane's four columns at a time,
// straight from the registers, every store touches 32 rows).  get(i, j, q): columns 32 i + 8 q + 4 h .. + 3 of the wave's
// block, row block j, packed.  out: row 0, column 0 of the tile; rows, cols: how much of it exists.  Chunk c of row r lies at
// c ^ (r & 15).
template <class T, class Get>
__device__ __forceinline__ void store_tile(char* lds, Get&& get, __bf16* out, long stride, long rows, long cols) {
  constexpr int CH = T::TM / 8;  // chunks of a row
  static_assert(T::TM * T::TN * 2 <= T::LDS && CH >= 16, "the results take the place of the operands");
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / T::WN, wn = wave % T::WN;
  __syncthreads();  // the tile's operands are done with
#pragma unroll
  for (int j = 0; j < T::NT; ++j) {
    const int r = (wn * T::NT + j) * 32 + l32;
#pragma unroll
    for (int i = 0; i < T::MT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = (wm * T::MT + i) * 4 + q;
        *reinterpret_cast<uint2*>(lds + (r * CH + (c ^ (r & 15))) * 16 + 8 * h) = get(i, j, q);
      }
  }
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

}  // namespace pdllm
