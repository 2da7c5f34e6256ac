// The vocabulary head for gfx950: z = h w^T from hidden states h [rows, D] and the head's weight w [V, D] (bf16), never
// written to memory.  Each workgroup forms a tile of logits on the matrix cores (gemm_core.h) and keeps of it what the
// call needs: the softmax statistics of its rows (maximum, sum, position of the maximum, logit of the label), which a
// small second kernel joins, or, for the gradient, the tile of softmax gradients that the two products behind it read.
//
//   logp[r] = -log(1 + exp(L - z[r, l])),  L = log sum over v != l of exp z[r, v]
//
// (the label's own term stays out of the sum: where the model is all but certain, 1 - p keeps its digits).
//   d[r, v] = -g[r] exp(z[r, v] - lse[r]) (v != l),  d[r, l] = -g[r] expm1(logp[r]);  grad_h = d w,  grad_w = d^T h.

#include "gemm_core.h"
#include "unmask_rule.h"

namespace pdllm {

constexpr float kLog2eH = 1.4426950408889634f;

struct HeadParams {
  const char* w;        // [V, D] bf16, row stride in bytes
  const char* h;        // [N, D]
  const char* last;     // [n_seqs, D] or NULL: the row in front of each block when the rows are read shifted by one
  long w_stride, h_stride, last_stride;  // bytes
  long V, N;
  int D;
  int block_len, shift;
  const long* labels;
  // tiles (see head_grid): n_full whole tiles, n_cut pieces of 64 rows of whole tiles, then the rows behind the whole columns
  int n_tok_tiles, n_voc_tiles, n_full, n_cut, rest_cols;
  // statistics
  float2* part;   // [N][parts]: maximum and sum over the part's entries (the label's excluded when labels are given)
  int* part_idx;  // [N][parts]: position of the maximum
  int parts;
  float* xlab;    // [N]: logit of the label
  int* joined;    // workgroups of the joining kernel that are done (cleared by this one), or NULL
  // gradient
  const float* lse;
  const float* logp;
  const float* g;
  __bf16* d;      // [N, ldd]: a piece of the softmax gradient, entries from v0 on
  long ldd;
  long v0;        // first entry of the piece; n_voc_tiles covers it
  char* hz;       // [N, D]: h with the rows of labels outside the vocabulary cleared (or NULL: an earlier piece did it)
  // few rows (np = their number rounded up to 32 or 64): d holds np rows, then np more with what its rounding left; a second
  // copy dt [entries][2 np] and hz [D][2 np] (every row of h twice) have the rows as the fast index
  __bf16* dt;
  int np;
};

// tile number -> tile: four neighbouring token tiles share a strip of the weight in the L2 of one XCD
__device__ __forceinline__ void head_tile(const HeadParams& p, int id, int& vt, int& nt) {
  const int per = 4 * p.n_voc_tiles;
  const int g = id / per;
  const int left = p.n_tok_tiles - 4 * g;
  const int width = left < 4 ? left : 4;
  const int r = id - g * per;
  vt = __builtin_amdgcn_readfirstlane(r / width);  // (a division leaves scalar registers)
  nt = __builtin_amdgcn_readfirstlane(4 * g + r - r / width * width);
}

template <class T>
__device__ __forceinline__ void head_logits(const HeadParams& p, int vt, long row0, Acc<T>& acc, char* lds) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned lds_base = (unsigned)(size_t)lds;
  const long v0 = p.v0 + (long)vt * T::TM;
  const unsigned kbytes = 2u * p.D;
  LoadKC<T::LA> la;
  la.init(p.w + v0 * p.w_stride, p.V - v0, (unsigned)p.w_stride, kbytes, wave, lane);
  LoadRows<T::LB> lb;
  lb.init(
      [&](unsigned row) __attribute__((always_inline)) {
        long t = row0 + row;
        t = t < p.N ? t : p.N - 1;
        if (p.shift) {
          const long b = t / p.block_len;
          if (t - b * p.block_len != 0) --t;
          else if (p.last) return p.last + b * p.last_stride;
        }
        return p.h + t * p.h_stride;
      },
      kbytes, wave, lane);
  mainloop_bf16<T, false, false>(
      acc, (int)(kbytes + KB - 1) / KB, lds_base, [&](int t, unsigned dst, auto copy) __attribute__((always_inline)) {
        constexpr int I = decltype(copy)::value;
        if constexpr (I < T::LA) la.template one<I>(t, dst + wave * (T::LA * 1024));
        else lb.template one<I - T::LA>(t, dst + T::A_BYTES + wave * (T::LB * 1024));
      });
}

struct Stat {
  float m, s;
  int idx;
};
__device__ __forceinline__ Stat stat_join(const Stat& a, const Stat& b) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  const float ref = r.m == -INFINITY ? 0.f : r.m;
  r.s = a.s * __builtin_amdgcn_exp2f((a.m - ref) * kLog2eH) + b.s * __builtin_amdgcn_exp2f((b.m - ref) * kLog2eH);
  const int ia = a.m == r.m ? a.idx : 0x7fffffff, ib = b.m == r.m ? b.idx : 0x7fffffff;
  r.idx = ia < ib ? ia : ib;
  return r;
}

// A tile of logits and its statistics per row: a lane's own values first (their maximum, then the sum of exp(x - max)), the other
// three lanes of the row, the other waves of the row.  Groups of up to 64 entries, whatever the tile: equal rows have equal
// statistics in tiles and in pieces of them, so that a tie between rows stays one.
template <class T, bool CONF>
__device__ __forceinline__ void head_stats_tile(const HeadParams& p, int vt, long row0, char* lds) {
  Acc<T> acc;
  head_logits<T>(p, vt, row0, acc, lds);

  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / T::WN, wn = wave % T::WN;
  const long vw = (long)vt * T::TM + wm * (32 * T::MT);  // first entry of the wave
  if (vw + 32 * T::MT > p.V) {                           // entries behind the vocabulary do not exist
#pragma unroll
    for (int i = 0; i < 2 * T::MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (vw + 16 * i + 4 * g + e >= p.V)
#pragma unroll
          for (int j = 0; j < 2 * T::NT; ++j) acc.v[i][j][e] = -INFINITY;
  }
  constexpr int GROUPS = T::MT > 2 ? T::MT / 2 : 1, BLOCKS = 2 * T::MT / GROUPS;
  static_assert(sizeof(Stat) * T::WM * GROUPS * T::TN <= T::LDS, "");
  __syncthreads();  // the tile's operands are done with: their place takes the statistics
#pragma unroll
  for (int j = 0; j < 2 * T::NT; ++j) {
    const int col = wn * (32 * T::NT) + 16 * j + l16;
    if constexpr (!CONF) {
      const long row = row0 + col;
      const long lab = row < p.N ? p.labels[row] : -1;
      const long rel = lab - vw;
      const bool mine = rel >= 0 && rel < 32 * T::MT && lab < p.V && ((rel >> 2) & 3) == g;
      if (__builtin_amdgcn_ballot_w64(mine) != 0) {
        const int at = mine ? (int)rel - 4 * g : -1;
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * T::MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (at == 16 * i + e) {
              x = acc.v[i][j][e];
              acc.v[i][j][e] = -INFINITY;
            }
        if (mine) p.xlab[row] = x;
      }
    }
#pragma unroll
    for (int q = 0; q < GROUPS; ++q) {
      float m = -INFINITY;
      int idx = 0x7fffffff;
#pragma unroll
      for (int i = q * BLOCKS; i < (q + 1) * BLOCKS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = acc.v[i][j][e];
          if constexpr (CONF) {
            if (x > m) idx = 16 * i + e;
          }
          m = fmaxf(m, x);
        }
      // the other lane groups hold the other entries of the same row
      const float m1 = fmaxf(m, __shfl_xor(m, 16, 64));
      const float top = half_swap_max(m1);
      const float ref = top == -INFINITY ? 0.f : top;
      float s = 0.f;
#pragma unroll
      for (int i = q * BLOCKS; i < (q + 1) * BLOCKS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s += __builtin_amdgcn_exp2f((acc.v[i][j][e] - ref) * kLog2eH);
      s += __shfl_xor(s, 16, 64);
      s = half_swap_sum(s);
      if constexpr (CONF) {
        // the lowest position among the lanes that hold the maximum
        int cand = m == top && idx != 0x7fffffff ? idx + 4 * g : 0x7fffffff;
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) {
          const int other = __shfl_xor(cand, o, 64);
          cand = other < cand ? other : cand;
        }
        idx = cand == 0x7fffffff ? cand : cand + (int)vw;
      }
      if (g == 0) reinterpret_cast<Stat*>(lds)[(wm * GROUPS + q) * T::TN + col] = {top, s, idx};
    }
  }
  __syncthreads();
  const int c = threadIdx.x;
  const long row = row0 + c;
  if (c < T::TN && row < p.N) {
    const Stat* sh = reinterpret_cast<const Stat*>(lds) + c;
    Stat a = sh[0];
#pragma unroll
    for (int q = 1; q < T::WM * GROUPS; ++q) a = stat_join(a, sh[q * T::TN]);
    const long o = row * p.parts + vt;
    p.part[o] = make_float2(a.m, a.s);
    if constexpr (CONF) p.part_idx[o] = a.idx;
  }
}

// A workgroup's tile: T for the whole tiles, then pieces of 64 rows (TS) of those that would be an almost empty last round of
// the compute units, and of the rows behind the last whole column.
template <class T, class TS, class F>
__device__ __forceinline__ void head_dispatch(const HeadParams& p, F&& tile) {
  int vt, nt;
  if ((int)blockIdx.x < p.n_full) {
    head_tile(p, xcd_remap(blockIdx.x, p.n_full), vt, nt);
    tile(static_cast<T*>(nullptr), vt, (long)nt * T::TN);
    return;
  }
  const int id = xcd_remap(blockIdx.x - p.n_full, gridDim.x - p.n_full);
  if (id < p.n_cut) {
    constexpr int Q = T::TN / TS::TN;
    head_tile(p, p.n_full + id / Q, vt, nt);
    tile(static_cast<TS*>(nullptr), vt, (long)nt * T::TN + (id % Q) * TS::TN);
  } else {
    const int r = id - p.n_cut;
    vt = __builtin_amdgcn_readfirstlane(r / p.rest_cols);
    tile(static_cast<TS*>(nullptr), vt, (long)p.n_tok_tiles * T::TN + (r - vt * p.rest_cols) * TS::TN);
  }
}

// Bound by the weight's bytes up to 128 rows (152064 x 3584: 182 us for 32 rows, 6.0 TB/s; 214 us for 128, 5.1 TB/s), above by the
// matrix instructions and the card's power (4096 rows: 3.14 to 3.21 ms, 1.39 to 1.42 PFLOP/s with the statistics; a library product
// of the same size, which writes its logits, 3.11 ms).  Between, by what whole tiles leave empty: 290, 384 and 512 rows take 460 to 470 us.  Forming one tile after the other in 256 workgroups, the next tile's copies in flight during
// the statistics, was no faster (4096 rows 3.31 ms, 1000 rows x 50021 x 1032 116.7 us for 117.4).
template <class T, class TS, bool CONF>
__global__ __launch_bounds__(T::THREADS, 2) void head_stats_kernel(const HeadParams p) {
  __shared__ __attribute__((aligned(1024))) char lds[T::LDS > TS::LDS ? T::LDS : TS::LDS];
  if (CONF && p.joined && blockIdx.x == 0 && threadIdx.x == 0) *p.joined = 0;
  head_dispatch<T, TS>(p, [&](auto* t, int vt, long row0) __attribute__((always_inline)) {
    head_stats_tile<std::remove_pointer_t<decltype(t)>, CONF>(p, vt, row0, lds);
  });
}

// Joins the parts of a row in a fixed order: a workgroup's 256 threads for one row, or a wave where a row has few parts.  The parts of
// a row lie side by side and are fetched four at a time by a thread (32 rows x 1188 parts: 12.8 us with the parts of 16
// rows interleaved and one fetch after the other, 7.9 us so).
struct UnmaskParams {
  long* block_ids;  // NULL: no transfer
  long n_seqs, block_len, mask_token_id;
  float threshold;
  uint8_t* transfer;
  int* n_left;
  int* joined;
};

template <bool CONF>
__global__ __launch_bounds__(256) void head_join_kernel(const float2* __restrict__ part, const int* __restrict__ part_idx,
                                                         const float* __restrict__ xlab, const long* __restrict__ labels,
                                                         int parts, long N, long V, float* out, float* __restrict__ lse_out,
                                                         long* token_out, const UnmaskParams un) {
  __shared__ Stat sh[4];
  const int per = parts > 256 ? 256 : 64;  // threads of a row
  const int at = threadIdx.x & (per - 1);
  const long row = (long)blockIdx.x * (256 / per) + threadIdx.x / per;
  Stat a = {-INFINITY, 0.f, 0x7fffffff};
  if (row < N) {
    const float2* v = part + row * parts;
    const int* vi = part_idx + row * parts;
    for (int q = at; q < parts; q += 4 * per) {
      float2 x[4];
      int idx[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool on = q + per * u < parts;
        x[u] = v[on ? q + per * u : q];
        idx[u] = CONF ? vi[on ? q + per * u : q] : 0;
        if (!on) x[u] = make_float2(-INFINITY, 0.f);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) a = stat_join(a, {x[u].x, x[u].y, idx[u]});
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const Stat b = {__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64), __shfl_xor(a.idx, o, 64)};
    a = stat_join(a, b);
  }
  if (per == 256) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a;
    __syncthreads();
    a = sh[0];
    for (int q = 1; q < 4; ++q) a = stat_join(a, sh[q]);
  }
  const bool writes = at == 0 && row < N;
  if constexpr (CONF) {
    if (writes) {
      out[row] = a.s == 0.f ? NAN : 1.f / a.s;           // every entry -inf: as softmax has it
      token_out[row] = a.idx == 0x7fffffff ? 0 : a.idx;  // a row of -inf and NaN alone has no maximum
    }
    if (!un.block_ids) return;
    // the workgroup that is done last makes the step's transfers (its order decides nothing: it sees every row's result)
    __shared__ int last;
    if (writes) __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(un.joined, 1) == (int)gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    for (long b = threadIdx.x >> 6; b < un.n_seqs; b += 4)
      unmask_block(out, token_out, un.block_ids, b, un.block_len, un.mask_token_id, un.threshold, un.transfer, un.n_left);
  } else {
    if (!writes) return;
    const float L = a.m + logf(a.s);
    const long lab = labels[row];
    if (lab < 0 || lab >= V) {
      out[row] = -INFINITY;
      if (lse_out) lse_out[row] = L;
    } else {
      const float x = xlab[row];
      const float d = L - x;
      float lp = -(fmaxf(d, 0.f) + log1pf(expf(-fabsf(d))));
      if (x == INFINITY || (x == -INFINITY && L == -INFINITY)) lp = NAN;
      out[row] = lp;
      // log(exp L + exp x), not x - logp: that loses digits where the label is far below the others, and is NaN at -inf
      if (lse_out) lse_out[row] = L == x ? L + 0.69314718f : fmaxf(L, x) + log1pf(expf(-fabsf(d)));
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------
// gradient
// ------------------------------------------------------------------------------------------------------------------

// One piece of the softmax gradient, rounded to bf16 as the operand of the two products behind it (each entry off by at
// most 2^-8 of itself: the gradients' errors are 0.0024 of their norm, the result's own rounding to bf16 alone 0.0017).  For few rows,
// where few entries make up a result and the products wait for memory anyway, the remainder of the rounding is kept beside it;
// above it would be a second product of the same size.  4096 rows x 32768 entries x 3584: 740 us, 1.30 PFLOP/s.
template <class T, bool FEW>
__device__ __forceinline__ void head_dlogits_tile(const HeadParams& p, int vt, long row0, char* lds) {
  Acc<T> acc;
  head_logits<T>(p, vt, row0, acc, lds);
  const int lane = threadIdx.x & 63, l16 = lane & 15, g4 = 4 * (lane >> 4);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / T::WN, wn = wave % T::WN;
  const int v_wave = wm * (32 * T::MT), r_wave = wn * (32 * T::NT);
  const long vl = (long)vt * T::TM + v_wave;                                        // first entry of the wave, in the piece
  const long left = p.V - p.v0 - vl;                                               // entries of the vocabulary from there on
  const int end = left < 0 ? 0 : left < 32 * T::MT ? (int)left : 32 * T::MT;
#pragma unroll
  for (int j = 0; j < 2 * T::NT; ++j) {
    const long row = row0 + r_wave + 16 * j + l16;
    const long lab = row < p.N ? p.labels[row] : -1;
    const bool in = lab >= 0 && lab < p.V;
    const float lse = in ? p.lse[row] : 0.f, g = in ? p.g[row] : 0.f;
#pragma unroll
    for (int i = 0; i < 2 * T::MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = -g * __builtin_amdgcn_exp2f((acc.v[i][j][e] - lse) * kLog2eH);
        acc.v[i][j][e] = in ? y : 0.f;  // (a row without a label may hold anything)
      }
    const long rel = lab - p.v0 - vl;
    const bool mine = in && rel >= 0 && rel < 32 * T::MT && ((int)rel & 12) == g4;
    if (__builtin_amdgcn_ballot_w64(mine) != 0) {
      const int at = mine ? (int)rel - g4 : -1;
      const float y = mine ? -g * expm1f(p.logp[row]) : 0.f;
#pragma unroll
      for (int i = 0; i < 2 * T::MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (at == 16 * i + e) acc.v[i][j][e] = y;
    }
  }
  if (end < 32 * T::MT) {  // entries behind the vocabulary: zeros, which the products read
#pragma unroll
    for (int i = 0; i < 2 * T::MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (16 * i + g4 + e >= end)
#pragma unroll
          for (int j = 0; j < 2 * T::NT; ++j) acc.v[i][j][e] = 0.f;
  }
  const long o = row0 * p.ldd + (long)vt * T::TM;
  store_acc<T>(lds, acc, [](float a, float b) __attribute__((always_inline)) { return pack_bf16x2(a, b); }, p.d + o, p.ldd, p.N - row0, T::TM);
  if constexpr (FEW) {
    // the remainder of a rounded pair
    auto low = [](float a, float b) __attribute__((always_inline)) {
      const unsigned w = pack_bf16x2(a, b);
      return pack_bf16x2(a - __uint_as_float(w << 16), b - __uint_as_float(w & 0xffff0000u));
    };
    store_acc<T>(lds, acc, low, p.d + p.np * p.ldd + o, p.ldd, p.N, T::TM);
    // the same with the rows as the fast index, through LDS: [entries of the tile][2 np], 16 bytes behind each
    const int pitch = 4 * p.np + 16;
    static_assert(T::TN == 64 && T::TM * (4 * 64 + 16) <= T::LDS, "");
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2 * T::NT; ++j) {
      const int r = r_wave + 16 * j + l16;
      if (r >= p.np) break;
#pragma unroll
      for (int i = 0; i < 2 * T::MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float x = acc.v[i][j][e], y = acc.v[i][j][e + 1];
          const unsigned h = pack_bf16x2(x, y), l = low(x, y);
          char* at = lds + (v_wave + 16 * i + g4 + e) * pitch + 2 * r;
          *reinterpret_cast<unsigned short*>(at) = (unsigned short)h;
          *reinterpret_cast<unsigned short*>(at + pitch) = (unsigned short)(h >> 16);
          *reinterpret_cast<unsigned short*>(at + 2 * p.np) = (unsigned short)l;
          *reinterpret_cast<unsigned short*>(at + pitch + 2 * p.np) = (unsigned short)(l >> 16);
        }
    }
    __syncthreads();
    const int chunks = p.np / 4;  // of a row
    char* dt = reinterpret_cast<char*>(p.dt + (long)vt * T::TM * (2 * p.np));
    for (int k = threadIdx.x; k < T::TM * chunks; k += T::THREADS)
      *reinterpret_cast<uint4*>(dt + 16L * k) = *reinterpret_cast<const uint4*>(lds + k / chunks * pitch + k % chunks * 16);
  }
}

template <class T, class TS, bool FEW>
__global__ __launch_bounds__(T::THREADS, 2) void head_dlogits_kernel(const HeadParams p) {
  __shared__ __attribute__((aligned(1024))) char lds[T::LDS > TS::LDS ? T::LDS : TS::LDS];
  if (p.hz) {
    // grad_w must not see the rows without a label (their states may hold anything): a copy with those rows cleared
    const int chunks = p.D / 8;
    const long rows = FEW ? p.np : p.N;
    for (long i = (long)blockIdx.x * T::THREADS + threadIdx.x; i < rows * chunks; i += (long)gridDim.x * T::THREADS) {
      const long r = FEW ? i % p.np : i / chunks;
      const int c = (int)(FEW ? i / p.np : i - r * chunks);
      const long lab = !FEW || r < p.N ? p.labels[r] : -1;
      uint4 v = {0, 0, 0, 0};
      if (lab >= 0 && lab < p.V) v = *reinterpret_cast<const uint4*>(p.h + r * p.h_stride + 16 * c);
      if constexpr (FEW) {
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
        unsigned short* o = reinterpret_cast<unsigned short*>(p.hz) + (long)c * 8 * (2 * p.np) + r;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e * 2 * p.np] = o[e * 2 * p.np + p.np] = (unsigned short)(w[e >> 1] >> (16 * (e & 1)));
      } else {
        *reinterpret_cast<uint4*>(p.hz + i * 16) = v;
      }
    }
  }
  head_dispatch<T, TS>(p, [&](auto* t, int vt, long row0) __attribute__((always_inline)) {
    head_dlogits_tile<std::remove_pointer_t<decltype(t)>, FEW>(p, vt, row0, lds);
  });
}

struct GradParams {
  const char* w;   // rows of the weight from the piece's first on
  const char* hz;  // [N, D], few rows: [D][2 np]
  const char* d;   // [N, ldd], few rows: [2 np, ldd]
  const char* dt;  // few rows: [entries][2 np]
  long w_stride, ldd;  // bytes
  long N;
  long vp;         // entries of the piece
  int D;
  int m_tiles, n_tiles, splits;  // of grad_h: column tiles, row tiles, splits of the entries
  int w_tiles;                   // of grad_w: column tiles
  int v_per;                     // of grad_w of few rows: entries of a wave
  long k_per;      // entries per split, a multiple of 64
  float* acc;      // [splits][N][D]
  __bf16* gh;      // written directly when the one split of the one piece is all of the sum
  long gh_stride;  // elements
  int add;         // the accumulators hold earlier pieces
  __bf16* gw;      // rows of grad_w from the piece's first on
  long gw_stride;  // elements
};

// grad_h of a piece: acc[split][row][c] (+)= sum over the split's entries of d[row][v] w[v][c].  Few rows: the tile holds all of them
// and behind them the remainders' rows, whose results a lane has beside the others.
template <class T, bool FEW>
__device__ __forceinline__ void head_grad_h_tile(const GradParams& p, int c0, long r0, int split, char* lds) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / T::WN, wn = wave % T::WN;
  const unsigned lds_base = (unsigned)(size_t)lds;
  const long k0 = split * p.k_per;
  long kn = p.vp - k0;
  kn = kn < 0 ? 0 : (kn < p.k_per ? kn : p.k_per);  // (a last, shorter piece may leave a split without entries)
  constexpr int SK = KB / 2;  // entries per stage
  const int steps = (int)((kn + SK - 1) / SK);
  const unsigned cols = 2u * (unsigned)(p.D - c0 < T::TM ? p.D - c0 : T::TM);
  LoadKS<T::LA, T::TM> la;
  la.init(p.w + k0 * p.w_stride + 2 * c0, p.w_stride, kn, cols, wave, lane);
  LoadKC<T::LB> lb;
  const unsigned kb = (unsigned)KB * steps;  // d is padded with zeros to whole stages
  const char* d0 = p.d + r0 * p.ldd + 2 * k0;
  lb.init(d0, FEW ? T::TN : p.N - r0, (unsigned)p.ldd, kb, wave, lane);
  Acc<T> acc;
  mainloop_bf16<T, true, false>(
      acc, steps, lds_base, [&](int t, unsigned dst, auto copy) __attribute__((always_inline)) {
        constexpr int I = decltype(copy)::value;
        if constexpr (I < T::LA) la.template one<I>(t, dst + wave * (T::LA * 1024));
        else lb.template one<I - T::LA>(t, dst + T::A_BYTES + wave * (T::LB * 1024));
      });
#pragma unroll
  for (int j = 0; j < (FEW ? T::NT : 2 * T::NT); ++j) {
    const long row = r0 + wn * (32 * T::NT) + 16 * j + l16;
    if (row >= p.N) continue;
    float* out = p.acc + ((long)split * p.N + row) * p.D;
#pragma unroll
    for (int i = 0; i < 2 * T::MT; ++i) {
      const int c = c0 + wm * (32 * T::MT) + 16 * i + 4 * g;
      if (c >= p.D) continue;
      f32x4 v = acc.v[i][j];
      if constexpr (FEW) v += acc.v[i][j + T::NT];
      if (p.gh) {
        *reinterpret_cast<uint2*>(p.gh + row * p.gh_stride + c) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        continue;
      }
      if (p.add) v += *reinterpret_cast<const f32x4*>(out + c);
      *reinterpret_cast<f32x4*>(out + c) = v;
    }
  }
}

// grad_h = the splits' accumulators, added in order, rounded once
__global__ __launch_bounds__(256) void head_grad_h_join_kernel(const float* __restrict__ acc, int splits, long N, int D,
                                                               __bf16* __restrict__ out, long stride) {
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= N * D) return;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; s += 4) {
    f32x4 a[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) a[u] = *reinterpret_cast<const f32x4*>(acc + (long)(s + u < splits ? s + u : s) * N * D + i);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (s + u < splits) v += a[u];
  }
  const long r = i / D;
  const uint2 w = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
  *reinterpret_cast<uint2*>(out + r * stride + (i - r * D)) = w;
}

// grad_w, the rows of a piece: gw[v][c] = sum over rows r of d[r][v] hz[r][c]
template <class T>
__device__ __forceinline__ void head_grad_w_tile(const GradParams& p, int c0, long v0, char* lds) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned lds_base = (unsigned)(size_t)lds;
  constexpr int SK = KB / 2;  // rows per stage
  const int steps = (int)((p.N + SK - 1) / SK);
  const unsigned cols = 2u * (unsigned)(p.D - c0 < T::TM ? p.D - c0 : T::TM);
  LoadKS<T::LA, T::TM> la;
  la.init(p.hz + 2 * c0, 2L * p.D, p.N, cols, wave, lane);
  LoadKS<T::LB, T::TN> lb;
  lb.init(p.d + 2 * v0, p.ldd, p.N, 2u * T::TN, wave, lane);  // the rows of d are whole tiles long
  Acc<T> acc;
  mainloop_bf16<T, true, true>(
      acc, steps, lds_base, [&](int t, unsigned dst, auto copy) __attribute__((always_inline)) {
        constexpr int I = decltype(copy)::value;
        if constexpr (I < T::LA) la.template one<I>(t, dst + wave * (T::LA * 1024));
        else lb.template one<I - T::LA>(t, dst + T::A_BYTES + wave * (T::LB * 1024));
      });
  store_acc<T>(lds, acc, [](float a, float b) __attribute__((always_inline)) { return pack_bf16x2(a, b); }, p.gw + v0 * p.gw_stride + c0,
               p.gw_stride, p.vp - v0, p.D - c0);
}

// Both products of a piece in one launch: the tiles of grad_h first (few, with the whole piece to sum over), those of grad_w
// (many, with the rows to sum over) fill the compute units they leave.
// The small tiles (80 KB of LDS, at most 128 registers) leave room for two workgroups on a compute unit, which hide each other's
// start and end: with few rows a tile of grad_w is a few stages and then 32 KB of results.
// 4096 rows x 32768 entries x 3584: 1454 us, 1.32 PFLOP/s, bound as the statistics are.
// The last strip of up to half a tile's columns takes tiles of half the width (TN): the gradient of 1000 rows x 50021 entries x 1032 364
// instead of 370 us, of 600 x 60000 x 520 190 instead of 196.
template <class TH, class TW, class TN>
__global__ __launch_bounds__(TW::THREADS, TW::MT * TW::NT <= 2 ? 4 : 2) void head_grad_kernel(const GradParams p) {
  static_assert(TH::THREADS == TW::THREADS && TN::THREADS == TW::THREADS && TN::LDS <= TW::LDS, "");
  constexpr bool NARROW = TN::TM < TW::TM;
  static_assert(!NARROW || (TN::TN == TH::TN && TN::TN == TW::TN && 2 * TN::TM == TH::TM && TH::TM == TW::TM), "");
  __shared__ __attribute__((aligned(1024))) char lds[TH::LDS > TW::LDS ? TH::LDS : TW::LDS];
#ifdef __HIP_DEVICE_COMPILE__  // (the host compiler cannot resolve the calls: their lambdas hold buffer descriptors)
  const int n_h = p.m_tiles * p.n_tiles * p.splits;
  if ((int)blockIdx.x < n_h) {
    const int id = xcd_remap(blockIdx.x, n_h);
    const int c0 = __builtin_amdgcn_readfirstlane(id % p.m_tiles) * TH::TM;
    const long r0 = (long)__builtin_amdgcn_readfirstlane((id / p.m_tiles) % p.n_tiles) * TH::TN;
    const int split = __builtin_amdgcn_readfirstlane(id / (p.m_tiles * p.n_tiles));
    if (NARROW && p.D - c0 <= TN::TM) head_grad_h_tile<TN, false>(p, c0, r0, split, lds);
    else head_grad_h_tile<TH, false>(p, c0, r0, split, lds);
  } else {
    const int id = xcd_remap(blockIdx.x - n_h, gridDim.x - n_h);
    const int c0 = __builtin_amdgcn_readfirstlane(id % p.w_tiles) * TW::TM;
    const long v0 = (long)__builtin_amdgcn_readfirstlane(id / p.w_tiles) * TW::TN;
    if (NARROW && p.D - c0 <= TN::TM) head_grad_w_tile<TN>(p, c0, v0, lds);
    else head_grad_w_tile<TW>(p, c0, v0, lds);
  }
#endif
}

// grad_w of few rows: 2 np products for each result, so the call waits for its results to be written.  Each wave keeps its
// columns of h in registers and goes through its entries by itself, 16 at a time: one fragment of d, the products, a
// store of 8 columns a lane (block 2 q holds columns 32 q + 8 g + e, e < 4, in lane group g, block 2 q + 1 those four further on).
constexpr int kFewColumns = 64;  // of a wave (128, with half the waves' registers for them, were no faster)
template <int NT>
__device__ __forceinline__ void head_grad_w_few(const GradParams& p, long id) {
  constexpr int C = kFewColumns, BLOCKS = C / 16, ROW = 64 * NT;  // bytes of a row of hz and dt
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int ct = __builtin_amdgcn_readfirstlane((int)(id % p.w_tiles));
  const long v0 = (long)__builtin_amdgcn_readfirstlane((int)(id / p.w_tiles)) * p.v_per;
  const long v1 = v0 + p.v_per < p.vp ? v0 + p.v_per : p.vp;
  if (v0 >= p.vp) return;
  const int c0 = ct * C;
  bf16x8 a[BLOCKS][NT];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) {
    const int c = c0 + 32 * (b / 2) + 8 * (l16 >> 2) + 4 * (b & 1) + (l16 & 3);
    const char* at = p.hz + (long)(c < p.D ? c : p.D - 1) * ROW + 16 * g;
#pragma unroll
    for (int k = 0; k < NT; ++k) a[b][k] = *reinterpret_cast<const bf16x8*>(at + 64 * k);
  }
  const char* src = p.dt + (v0 + l16) * ROW + 16 * g;
  bf16x8 d[NT], next[NT];
#pragma unroll
  for (int k = 0; k < NT; ++k) next[k] = *reinterpret_cast<const bf16x8*>(src + 64 * k);
  const bool wide = (((uintptr_t)p.gw | (uintptr_t)(2 * p.gw_stride)) & 15) == 0;
  for (long v = v0; v < v1; v += 16) {
#pragma unroll
    for (int k = 0; k < NT; ++k) d[k] = next[k];
    if (v + 16 < v1) {
      src += 16 * ROW;
#pragma unroll
      for (int k = 0; k < NT; ++k) next[k] = *reinterpret_cast<const bf16x8*>(src + 64 * k);
    }
    f32x4 acc[BLOCKS];
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
        acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[b][k], d[k], k == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[b], 0, 0, 0);
    if (v + l16 >= v1) continue;
    __bf16* out = p.gw + (v + l16) * p.gw_stride + c0 + 8 * g;
#pragma unroll
    for (int q = 0; q < BLOCKS / 2; ++q) {
      if (c0 + 32 * q + 8 * g >= p.D) continue;
      const uint4 w = {pack_bf16x2(acc[2 * q][0], acc[2 * q][1]), pack_bf16x2(acc[2 * q][2], acc[2 * q][3]),
                       pack_bf16x2(acc[2 * q + 1][0], acc[2 * q + 1][1]), pack_bf16x2(acc[2 * q + 1][2], acc[2 * q + 1][3])};
      if (wide) {
        *reinterpret_cast<uint4*>(out + 32 * q) = w;
      } else {
        *reinterpret_cast<uint2*>(out + 32 * q) = {w.x, w.y};
        *reinterpret_cast<uint2*>(out + 32 * q + 4) = {w.z, w.w};
      }
    }
  }
}

// Both products of up to 16 NT rows: tiles of grad_h, 256 columns x all rows and a share of the piece, then the waves of grad_w.
// Bound by the weight read and its gradient written: 32 rows x 126464 x 4096 485 us, 4.3 TB/s (a copy of 2 GiB reaches 4.9); with
// tiles of 128 x 128 through LDS for grad_w, two stages and 32 KB of results each, 600 to 710 us.
template <int NT>
__global__ __launch_bounds__(512, NT == 2 ? 4 : 2) void head_grad_few_kernel(const GradParams p) {
  typedef Tile<1, NT, 8, 1, 2> T;
  __shared__ __attribute__((aligned(1024))) char lds[T::LDS];
#ifdef __HIP_DEVICE_COMPILE__
  const int n_h = p.m_tiles * p.splits;
  if ((int)blockIdx.x < n_h) {
    const int id = xcd_remap(blockIdx.x, n_h);
    head_grad_h_tile<T, true>(p, __builtin_amdgcn_readfirstlane(id % p.m_tiles) * T::TM, 0, __builtin_amdgcn_readfirstlane(id / p.m_tiles), lds);
    return;
  }
  head_grad_w_few<NT>(p, 8L * xcd_remap(blockIdx.x - n_h, gridDim.x - n_h) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
#endif
}

// ------------------------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------------------------

namespace {

using TileL = Tile<4, 2, 2, 4, 2>;   // 256 entries x 256 rows, 8 waves
using TileR = Tile<2, 1, 4, 2, 3>;   // 256 x 64, 8 waves: pieces of 256 x 256
using TileM = Tile<2, 2, 4, 2, 3>;   // 256 x 128
using TileS2 = Tile<1, 2, 4, 1, 3>;  // 128 x 64, 4 waves
using TileS = Tile<1, 1, 4, 1, 4>;   // 128 x 32

constexpr long kMaxRows = 1L << 24;
constexpr long kMaxVocab = 1L << 30;

// Tiles of 128 x 64 where they are at most one round, two to a compute unit (us in tiles of 256 x 256 and so: 150 rows x 20000 x 3584
// 72 and 41, 100 x 16000 x 4096 42 and 36, 407 x 448 x 3096 33 and 27, 1024 x 4096 x 3584 44 and 43, 300 x 9000 x 2048 27 and 29)
bool small_tiles(long n, long v) { return n <= 64 || ((v + 127) / 128) * ((n + 63) / 64) <= 512; }

// parts of a row in the workspace: the vocabulary tiles
int stat_parts(long n, long v) {
  const int tm = small_tiles(n, v) ? TileS::TM : TileL::TM;
  static_assert(TileS::TM == TileS2::TM && TileM::TM == TileL::TM, "two heights of tiles");
  return (int)((v + tm - 1) / tm);
}

int64_t stats_ws(long n, long v, bool conf) { return (int64_t)stat_parts(n, v) * n * (conf ? 12 : 8) + (conf ? 4 : 4 * n); }

// The grid over n_voc_tiles x N rows: whole tiles of T; pieces of TS where an almost empty last round of the 256 compute units becomes
// one round of them (784 tiles of 1000 rows x 50021 entries x 3584: 335 us in four rounds, 297 in three and one of pieces; x 1032 127
// and 114; 594 tiles of 128 rows x 152064 x 3584: 222 and 215).  Up to 128 rows behind the last whole column are pieces too (2051
// rows x 126464 x 4096: 1793 us as a column of whole tiles, 1654 so; 640 x 50021 x 3584: 255 and 237); beside a single column, where
// reading the weight again counts, up to 64 and only if it stays in the last-level cache (300 x 50000 x 2048: 96 and 81; but 290 x
// 152064 x 3584 461 and 511, 384 x 152064 x 3584 467 and 575).
template <class T, class TS>
long head_grid(HeadParams& p) {
  constexpr int Q = T::TN / TS::TN;
  const long rest = p.N % T::TN;
  const bool again = p.N >= 2 * T::TN || (long)p.n_voc_tiles * T::TM * 2 * p.D <= (256L << 20);
  const bool cut_rest = Q > 1 && rest > 0 && again && rest <= (p.N >= 2 * T::TN ? T::TN / 2 : T::TN / 4);
  p.n_tok_tiles = (int)(p.N / T::TN + (rest > 0 && !cut_rest));
  p.rest_cols = cut_rest ? (int)((rest + TS::TN - 1) / TS::TN) : 0;
  const long whole = (long)p.n_voc_tiles * p.n_tok_tiles, last = whole % 256;
  const long full = Q > 1 && Q * last <= 256 ? whole - last : whole;
  const long grid = full + Q * (whole - full) + (long)p.n_voc_tiles * p.rest_cols;
  p.n_full = (int)full;
  p.n_cut = (int)(Q * (whole - full));
  return launch_fits(grid, T::THREADS) ? grid : -1;
}

template <class T, class TS, bool CONF>
int launch_stats(HeadParams& p, hipStream_t s) {
  p.n_voc_tiles = (int)((p.V + T::TM - 1) / T::TM);
  const long grid = head_grid<T, TS>(p);
  if (grid < 0) return PDLLM_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((head_stats_kernel<T, TS, CONF>), dim3((unsigned)grid), dim3(T::THREADS), 0, s, p);
  return launch_status();
}

int check_head(const void* hidden, int64_t h_stride, const void* weight, int64_t w_stride, int64_t n, int64_t v, int32_t d) {
  if (n < 0 || v <= 0 || d <= 0 || d % 8 || n > kMaxRows || v > kMaxVocab || d > (1 << 20)) return PDLLM_ERR_SHAPE;
  if (!weight || (!hidden && n > 0)) return PDLLM_ERR_NULL;
  if (h_stride < d || w_stride < d || h_stride % 8 || w_stride % 8) return PDLLM_ERR_STRIDE;
  if ((uintptr_t)hidden % 16 || (uintptr_t)weight % 16) return PDLLM_ERR_STRIDE;
  if (w_stride * 2 * 256 >= 0x7fffffffL) return PDLLM_ERR_STRIDE;  // a tile's rows lie within 31-bit offsets
  return PDLLM_OK;
}

template <bool CONF>
int stats(HeadParams& p, void* workspace, int64_t workspace_bytes, float* out, float* lse_out, long* token_out,
          UnmaskParams un, hipStream_t s) {
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < stats_ws(p.N, p.V, CONF)) return PDLLM_ERR_WORKSPACE;
  const int parts = p.parts = stat_parts(p.N, p.V);
  p.part = static_cast<float2*>(workspace);
  float* next = reinterpret_cast<float*>(p.part + (long)parts * p.N);
  p.part_idx = reinterpret_cast<int*>(next);
  p.xlab = next;
  if (un.block_ids) p.joined = un.joined = p.part_idx + (long)parts * p.N;
  const long joins = parts > 256 ? p.N : (p.N + 3) / 4;
  if (!launch_fits(joins, 256)) return PDLLM_ERR_UNSUPPORTED;
  int st;
  if (p.N <= 32) st = launch_stats<TileS, TileS, CONF>(p, s);
  else if (small_tiles(p.N, p.V)) st = launch_stats<TileS2, TileS2, CONF>(p, s);
  else if (p.N <= 128) st = launch_stats<TileM, TileR, CONF>(p, s);
  else st = launch_stats<TileL, TileR, CONF>(p, s);
  if (st != PDLLM_OK) return st;
  hipLaunchKernelGGL(head_join_kernel<CONF>, dim3((unsigned)joins), dim3(256), 0, s, p.part, p.part_idx, p.xlab,
                     p.labels, parts, p.N, p.V, out, lse_out, token_out, un);
  return launch_status();
}

// ---- gradient: sizes of the workspace's regions ----
// A piece of d, so that the workspace does not grow with the vocabulary; as large as the last-level cache, though not alone in it (of
// 4096 rows the products of a piece also read 235 MB of weight and write as much).  Smaller pieces mean more launches.
constexpr long kPieceBytes = 256L << 20;
constexpr long kMaxPiece = 1L << 21;        // 256 rows of a piece lie within 31-bit offsets
constexpr int kFewRows = 64;                // up to here the remainders are carried

struct GradPlan {
  int np, splits, small;  // np: rows of few, rounded up (or 0); small: the small tiles
  long vp;                // entries of a piece (a multiple of 256)
  int direct;             // grad_h needs no accumulators
  int64_t hz, d, dt, acc;  // bytes
};

int64_t align256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// Pieces as long as the workspace allows, up to kPieceBytes of d: of 4096 rows 32768 entries, 128 x 16 tiles of logits and 128 x 14 of
// grad_w (3584 columns), whole rounds of the 256 compute units.  have < 0: the size that is asked for.
bool plan_grad(long n, long v, int d, int64_t have, GradPlan& g) {
  g.np = n <= 32 ? 32 : n <= kFewRows ? 64 : 0;
  const long vall = (v + 255) / 256 * 256;
  // the small tiles where the sums over rows are short or the large ones would leave compute units idle
  g.small = n <= 256 || ((d + 255) / 256) * (vall / 256) < 192;
  const long tiles = ((d + 255) / 256) * (g.np ? 1 : g.small ? (n + 63) / 64 : (n + 255) / 256);
  const long slots = g.np == 64 || !g.small ? 256 : 512;  // workgroups at a time
  const long most = tiles < slots ? slots / tiles : 1;
  const long rows = g.np ? 2 * g.np : n;  // of d
  g.hz = align256(2L * rows * d);
  for (long piece = kPieceBytes / (2 * rows);; piece = g.vp / 2) {
    piece = piece < kMaxPiece ? piece : kMaxPiece;
    piece = piece >= 8192 ? piece / 4096 * 4096 : piece / 256 * 256;
    piece = piece < 256 ? 256 : (piece < vall ? piece : vall);
    // grad_h: enough splits of the piece for every compute unit, at least four stages each
    const long s = piece / 256;
    g.splits = (int)(s < 1 ? 1 : (s < most ? s : most));
    g.vp = piece;
    g.d = align256(2L * rows * piece);
    g.dt = g.np ? g.d : 0;
    // a short sum is not split: the launch that would join the splits costs more than 16 stages
    g.direct = piece >= vall && (g.splits == 1 || vall <= 1024);
    if (g.direct) g.splits = 1;
    g.acc = g.direct ? 0 : align256(4L * g.splits * n * d);
    if (have < 0 || g.hz + g.d + g.dt + g.acc <= have) return true;
    if (piece <= 256) return false;
  }
}

template <class T, class TS, bool FEW>
int launch_dlogits(HeadParams& p, hipStream_t s) {
  const long grid = head_grid<T, TS>(p);
  if (grid < 0) return PDLLM_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((head_dlogits_kernel<T, TS, FEW>), dim3((unsigned)grid), dim3(T::THREADS), 0, s, p);
  return launch_status();
}

using TileH = Tile<4, 2, 2, 4, 2>;  // grad_h, grad_w: 256 columns x 256 rows or entries
using TileN = Tile<2, 2, 2, 4, 2>;   // 128 columns x 256: the last strip
using TileH2 = Tile<1, 2, 8, 1, 2>;  // grad_h of small problems: 256 columns x 64 rows
using TileW2 = Tile<1, 2, 4, 2, 2>;  // grad_w of small problems: 128 columns x 128 entries

}  // namespace

}  // namespace pdllm

using namespace pdllm;

extern "C" int64_t pdllm_head_workspace_bytes(int64_t n_rows, int64_t vocab) {
  if (n_rows < 0 || vocab <= 0 || n_rows > kMaxRows || vocab > kMaxVocab) return PDLLM_ERR_SHAPE;
  if (n_rows == 0) return 0;
  const int64_t a = stats_ws(n_rows, vocab, true), b = stats_ws(n_rows, vocab, false);
  return a > b ? a : b;
}

extern "C" int pdllm_head_selfinfo_logprob(const void* hidden, int64_t hidden_stride, const void* weight,
                                           int64_t weight_stride, const int64_t* labels, int64_t n_rows, int64_t vocab,
                                           int32_t dim, void* workspace, int64_t workspace_bytes, float* logp_out,
                                           float* lse_out, pdllm_stream_t stream) {
  int st = check_head(hidden, hidden_stride, weight, weight_stride, n_rows, vocab, dim);
  if (st != PDLLM_OK || n_rows == 0) return st;
  if (!labels || !logp_out) return PDLLM_ERR_NULL;
  HeadParams p = {};
  p.w = static_cast<const char*>(weight);
  p.h = static_cast<const char*>(hidden);
  p.w_stride = 2 * weight_stride;
  p.h_stride = 2 * hidden_stride;
  p.V = vocab;
  p.N = n_rows;
  p.D = dim;
  p.block_len = 1;
  p.labels = reinterpret_cast<const long*>(labels);
  return stats<false>(p, workspace, workspace_bytes, logp_out, lse_out, nullptr, {}, static_cast<hipStream_t>(stream));
}

namespace pdllm {
namespace {

int conf_argmax(const void* hidden, int64_t hidden_stride, const void* last_hidden, int64_t last_hidden_stride,
                const void* weight, int64_t weight_stride, int64_t n_seqs, int64_t block_len, int64_t vocab, int32_t dim,
                int32_t shift, void* workspace, int64_t workspace_bytes, float* conf_out, int64_t* token_out,
                const UnmaskParams& un, pdllm_stream_t stream) {
  if (n_seqs < 0 || block_len <= 0 || block_len > kMaxRows || n_seqs > kMaxRows) return PDLLM_ERR_SHAPE;
  const int64_t n = n_seqs * block_len;
  int st = check_head(hidden, hidden_stride, weight, weight_stride, n, vocab, dim);
  if (st != PDLLM_OK || n == 0) return st;
  if (!conf_out || !token_out) return PDLLM_ERR_NULL;
  if (last_hidden && (last_hidden_stride < dim || last_hidden_stride % 8 || (uintptr_t)last_hidden % 16)) return PDLLM_ERR_STRIDE;
  HeadParams p = {};
  p.w = static_cast<const char*>(weight);
  p.h = static_cast<const char*>(hidden);
  p.last = static_cast<const char*>(last_hidden);
  p.w_stride = 2 * weight_stride;
  p.h_stride = 2 * hidden_stride;
  p.last_stride = 2 * last_hidden_stride;
  p.V = vocab;
  p.N = n;
  p.D = dim;
  p.block_len = (int)block_len;
  p.shift = shift ? 1 : 0;
  return stats<true>(p, workspace, workspace_bytes, conf_out, nullptr, reinterpret_cast<long*>(token_out), un,
                     static_cast<hipStream_t>(stream));
}

}  // namespace
}  // namespace pdllm

extern "C" int pdllm_head_conf_argmax(const void* hidden, int64_t hidden_stride, const void* last_hidden,
                                      int64_t last_hidden_stride, const void* weight, int64_t weight_stride, int64_t n_seqs,
                                      int64_t block_len, int64_t vocab, int32_t dim, int32_t shift, void* workspace,
                                      int64_t workspace_bytes, float* conf_out, int64_t* token_out, pdllm_stream_t stream) {
  return conf_argmax(hidden, hidden_stride, last_hidden, last_hidden_stride, weight, weight_stride, n_seqs, block_len, vocab, dim,
                     shift, workspace, workspace_bytes, conf_out, token_out, {}, stream);
}

extern "C" int pdllm_head_denoise_unmask(const void* hidden, int64_t hidden_stride, const void* last_hidden,
                                         int64_t last_hidden_stride, const void* weight, int64_t weight_stride,
                                         int64_t n_seqs, int64_t block_len, int64_t vocab, int32_t dim, int32_t shift,
                                         int64_t* block_ids, int64_t mask_token_id, float threshold, void* workspace,
                                         int64_t workspace_bytes, float* conf_out, int64_t* token_out, uint8_t* transfer_out,
                                         int32_t* n_masked_left, pdllm_stream_t stream) {
  if (n_seqs > 0 && (!block_ids || !transfer_out)) return PDLLM_ERR_NULL;
  // up to 32 blocks the last workgroup of the joining kernel makes the transfers (one launch less); more of them are quicker
  // done by a launch of their own
  UnmaskParams un = {};
  if (n_seqs <= 32) un = {reinterpret_cast<long*>(block_ids), (long)n_seqs, (long)block_len, (long)mask_token_id, threshold, transfer_out, n_masked_left, nullptr};
  const int st = conf_argmax(hidden, hidden_stride, last_hidden, last_hidden_stride, weight, weight_stride, n_seqs, block_len, vocab,
                             dim, shift, workspace, workspace_bytes, conf_out, token_out, un, stream);
  if (st != PDLLM_OK || n_seqs <= 32) return st;
  return pdllm_threshold_unmask(conf_out, token_out, block_ids, n_seqs, block_len, mask_token_id, threshold, transfer_out,
                                n_masked_left, stream);
}

extern "C" int64_t pdllm_head_selfinfo_grad_workspace_bytes(int64_t n_rows, int64_t vocab, int32_t dim) {
  if (n_rows < 0 || vocab <= 0 || dim <= 0 || dim % 8 || n_rows > kMaxRows || vocab > kMaxVocab || dim > (1 << 20))
    return PDLLM_ERR_SHAPE;
  if (n_rows == 0) return 0;
  GradPlan g;
  plan_grad(n_rows, vocab, dim, -1, g);
  return g.hz + g.d + g.dt + g.acc;
}

extern "C" int pdllm_head_selfinfo_grad(const void* hidden, int64_t hidden_stride, const void* weight, int64_t weight_stride,
                                        const int64_t* labels, const float* logp, const float* lse, const float* grad_logp,
                                        int64_t n_rows, int64_t vocab, int32_t dim, void* workspace, int64_t workspace_bytes,
                                        void* grad_hidden, int64_t grad_hidden_stride, void* grad_weight,
                                        int64_t grad_weight_stride, pdllm_stream_t stream) {
  int st = check_head(hidden, hidden_stride, weight, weight_stride, n_rows, vocab, dim);
  if (st != PDLLM_OK) return st;
  if (!grad_weight || (n_rows > 0 && (!labels || !logp || !lse || !grad_logp || !grad_hidden))) return PDLLM_ERR_NULL;
  if (grad_hidden_stride < dim || grad_hidden_stride % 4 || grad_weight_stride < dim || grad_weight_stride % 4 ||
      (uintptr_t)grad_hidden % 8 || (uintptr_t)grad_weight % 8)
    return PDLLM_ERR_STRIDE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (n_rows == 0) {  // a sum over no rows
    GradParams q = {};
    q.D = dim;
    q.w_tiles = (dim + 255) / 256;  // (no tiles of grad_h)
    const long tiles = q.w_tiles * ((vocab + 255) / 256);
    q.vp = vocab;
    q.gw = static_cast<__bf16*>(grad_weight);
    q.gw_stride = grad_weight_stride;
    if (!launch_fits(tiles, TileH::THREADS)) return PDLLM_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((head_grad_kernel<TileH, TileH, TileN>), dim3((unsigned)tiles), dim3(TileH::THREADS), 0, s, q);
    return launch_status();
  }
  GradPlan g;
  if (!workspace || (uintptr_t)workspace % 256 || !plan_grad(n_rows, vocab, dim, workspace_bytes, g)) return PDLLM_ERR_WORKSPACE;
  const long joins = (n_rows * (dim / 4) + 255) / 256;
  if (!g.direct && !launch_fits(joins, 256)) return PDLLM_ERR_UNSUPPORTED;
  char* ws = static_cast<char*>(workspace);
  HeadParams p = {};
  p.w = static_cast<const char*>(weight);
  p.h = static_cast<const char*>(hidden);
  p.w_stride = 2 * weight_stride;
  p.h_stride = 2 * hidden_stride;
  p.V = vocab;
  p.N = n_rows;
  p.D = dim;
  p.block_len = 1;
  p.labels = reinterpret_cast<const long*>(labels);
  p.lse = lse;
  p.logp = logp;
  p.g = grad_logp;
  p.d = reinterpret_cast<__bf16*>(ws + g.hz);
  p.dt = reinterpret_cast<__bf16*>(ws + g.hz + g.d);
  p.np = g.np;
  p.ldd = g.vp;
  GradParams q = {};
  q.hz = ws;
  q.d = ws + g.hz;
  q.dt = ws + g.hz + g.d;
  q.w_stride = p.w_stride;
  q.ldd = 2 * g.vp;
  q.N = n_rows;
  q.D = dim;
  q.m_tiles = (dim + 255) / 256;
  const bool few = g.np != 0;
  static_assert(TileW2::TM == TileW2::TN && TileH::TM == TileH::TN, "square tiles");
  const int tw = few ? kFewColumns : g.small ? TileW2::TM : TileH::TM;
  q.w_tiles = (dim + tw - 1) / tw;
  q.n_tiles = (int)(few ? 1 : g.small ? (n_rows + TileH2::TN - 1) / TileH2::TN : (n_rows + TileH::TN - 1) / TileH::TN);
  q.acc = reinterpret_cast<float*>(ws + g.hz + g.d + g.dt);
  q.gw_stride = grad_weight_stride;
  q.gh = g.direct ? static_cast<__bf16*>(grad_hidden) : nullptr;
  q.gh_stride = grad_hidden_stride;
  for (long v0 = 0; v0 < vocab; v0 += g.vp) {
    const long vp = vocab - v0 < g.vp ? vocab - v0 : g.vp;
    p.v0 = v0;
    p.hz = v0 == 0 ? ws : nullptr;
    const int tm = small_tiles(n_rows, vp) ? TileS2::TM : TileL::TM;
    p.n_voc_tiles = (int)((vp + tm - 1) / tm);
    st = few ? launch_dlogits<TileS2, TileS2, true>(p, s)
         : tm == TileS2::TM ? launch_dlogits<TileS2, TileS2, false>(p, s) : launch_dlogits<TileL, TileR, false>(p, s);
    if (st != PDLLM_OK) return st;
    q.w = p.w + v0 * p.w_stride;
    q.vp = vp;
    q.add = v0 > 0;
    q.splits = g.splits;
    q.k_per = ((vp + g.splits - 1) / g.splits + 63) / 64 * 64;
    q.gw = static_cast<__bf16*>(grad_weight) + v0 * grad_weight_stride;
    // few rows: 512 entries to a wave (8 or 16 KB of h read for 64 KB of results), fewer where the card would not be full
    q.v_per = q.w_tiles * ((vp + 511) / 512) >= 4096 ? 512 : 64;
    const long n_w = few ? (q.w_tiles * ((vp + q.v_per - 1) / q.v_per) + 7) / 8 : q.w_tiles * ((vp + tw - 1) / tw);
    const long grid = (long)q.m_tiles * q.n_tiles * q.splits + n_w;
    if (!launch_fits(grid, 512)) return PDLLM_ERR_UNSUPPORTED;
    const dim3 blocks((unsigned)grid), threads(512);
    if (g.np == 32) hipLaunchKernelGGL(head_grad_few_kernel<2>, blocks, threads, 0, s, q);
    else if (g.np == 64) hipLaunchKernelGGL(head_grad_few_kernel<4>, blocks, threads, 0, s, q);
    else if (g.small) hipLaunchKernelGGL((head_grad_kernel<TileH2, TileW2, TileW2>), blocks, threads, 0, s, q);
    else hipLaunchKernelGGL((head_grad_kernel<TileH, TileH, TileN>), blocks, threads, 0, s, q);
    if ((st = launch_status()) != PDLLM_OK) return st;
  }
  if (g.direct) return PDLLM_OK;
  hipLaunchKernelGGL(head_grad_h_join_kernel, dim3((unsigned)joins), dim3(256), 0, s, q.acc, g.splits, n_rows, dim,
                     static_cast<__bf16*>(grad_hidden), grad_hidden_stride);
  return launch_status();
}
