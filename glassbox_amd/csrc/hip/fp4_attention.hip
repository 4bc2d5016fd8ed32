// Attention over four-bit pages (fp4.h): o = sum_t softmax_t(scale q . k_t) v_t over the keys t of a request up to the row's own
// position (and, with a window, not further back), for the grouped query heads of rows of any number a request.
//
// The columns of a (request, kv head) are its rows' heads, column c the head c % rep of row c / rep: whatever the grouping, they fill
// the 16 columns of a matrix-core tile without gaps.  A wave holds 16 R columns and goes over the keys 64 at a time:
//
//   scores   S[t, c] = K[t, :] . Q[:, c], 16 x 16 x 32 products.  K is the left operand: lane (r, g) = (l % 16, l / 16) takes token
//            16 (r / 4) + 4 j + r % 4 in tile j and of each run of four blocks the block g (blocks of 16 or 8 channels where a head has
//            fewer): with 128 channels its 32 channels are 16 bytes and one scale, and the scales of j = 0..3 one word.  Which
//            channels a lane multiplies is free, as long as Q is laid out alike.
//   softmax  lane (r, g) then holds of column r the tokens 16 g + 4 j + x: 16 consecutive ones.  Running maximum and sum, in 32 bits.
//   sums     O[d, c] += V[d, t] . P[t, c]: P is the right operand as it lies in the registers; a lane's 16 tokens of V's channels
//            (r, r + 16) of a block are 16 consecutive bytes, and their scales 16 more.
//
// Codes become bf16 in registers, two an instruction with their scale, exactly; nothing passes through LDS but the joining of waves.
// A row of 32 bits counts as three bf16 terms (fp4.h), and so do its probabilities.  Those of a bf16 row count as two, off by 2^-16: its
// result is rounded once, at the end.  (As one term they were off by 2^-8: the distance from the 64-bit definition was 0.0021 of the results where their
// own rounding is 0.0016, and far more of sums that cancel; it takes 3 to 9 % less time for single tokens, 9 to 16 % less for portions.)
//
// Few columns (decoding): the waves of a workgroup share out the tiles and are joined through LDS; a long context is cut into runs
// for several workgroups, joined by a second kernel.  More columns: each wave has columns of its own and all of a run's keys.
#include "fp4.h"

#include <algorithm>
#include <cmath>

namespace gb {

constexpr int kTile = 64;        // keys a wave takes at a time
constexpr float kLargest = 3.402823466e38f;
constexpr int kMostSplits = 64;  // runs of a context: a lane each in the kernel that joins them

struct AttendArgs {
  const void* q;
  void* out;
  const int32_t *q_start, *q_len, *pos0, *tables;
  const uint8_t *k, *v;
  float* acc;
  float2* ml;
  int q_stride, out_stride, n, table_stride, table_cols, pages, nkv, rep, page, page_shift, max_q, window, chunk, splits, col_tiles;
  float scale;   // of the scores, times log2 e
  int q_wide, out_wide;
};

// how a lane's channels lie: units of 32, 16 or 8 channels, unit g + 4 i of the head
template <int NB> struct Units {
  static constexpr int kChannels = NB % 4 == 0 ? 32 : NB % 2 == 0 ? 16 : 8;
  static constexpr int kWords = kChannels / 8;
  static constexpr int kCount = NB / kWords;   // units a lane: NB words in all
};

__device__ __forceinline__ float quads_max(float v) {   // over the four lanes of a column
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t w = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// 0x80 in each byte that is 255
__device__ __forceinline__ uint32_t bytes_255(uint32_t w) {
  const uint32_t t = ~w;
  return ~(((t & 0x7f7f7f7fu) + 0x7f7f7f7fu) | t | 0x7f7f7f7fu);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

template <typename T> __device__ __forceinline__ void store4(T* p, bool wide, const float (&x)[4]) {
  if constexpr (std::is_same_v<T, float>) {
    if (wide) {
      *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
      return;
    }
  } else {
    if (wide) {
      *reinterpret_cast<bf16x4*>(p) = bf16x4{(bf16)x[0], (bf16)x[1], (bf16)x[2], (bf16)x[3]};
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = (T)x[i];
}

// ---- what both kernels do ------------------------------------------------------------------------------------------------------
// the page numbers of 16 tokens of keys and 16 of values of a lane, and where in their pages these begin
struct Places {
  int kp, vp, koff, voff;
};
__device__ __forceinline__ Places look_up(const AttendArgs& a, const int32_t* table, uint32_t kt, uint32_t vt) {
  const uint32_t page = a.page, columns = a.table_cols;   // (whatever the tokens' numbers, what is read lies in the table)
  const uint32_t ki = a.page_shift >= 0 ? kt >> a.page_shift : kt / page, vi = a.page_shift >= 0 ? vt >> a.page_shift : vt / page;
  const int k0 = table[min(ki, columns - 1)], v0 = table[min(vi, columns - 1)];
  return {ki < columns ? k0 : -1, vi < columns ? v0 : -1, (int)(kt - ki * page), (int)(vt - vi * page)};
}
// the first key that a window leaves a position; no sum passes 32 bits, whatever the position
__device__ __forceinline__ int window_from(const AttendArgs& a, int pos) { return a.window > 0 ? max(pos, a.window - 1) - (a.window - 1) : 0; }
// What a column's sum of p v is multiplied by: zeros for one that sees no key (its maximum is still minus infinity), NaN for one all of whose
// keys have scores of minus infinity.
__device__ __forceinline__ float over_sum(float sum, float m) { return sum > 0.f || sum != sum ? 1.f / sum : m == -__builtin_inff() ? 0.f : __builtin_nanf(""); }
// a page of the pool; page 0 in the place of any other number, which is not read
__device__ __forceinline__ bool known_page(const AttendArgs& a, int page) { return (unsigned)page < (unsigned)a.pages; }
__device__ __forceinline__ size_t page_at(const AttendArgs& a, int page, int kvh, size_t head_bytes) {
  return ((size_t)(known_page(a, page) ? page : 0) * a.nkv + kvh) * head_bytes;
}

// the query of a column, its channels as the lanes take those of the keys
template <typename T, int NB> __device__ __forceinline__ void load_query(const T* row, int g, bool wide, bf16x8 (&qf)[kFp4Terms<T>][NB]) {
  using U = Units<NB>;
#pragma unroll
  for (int i = 0; i < U::kCount; ++i)
#pragma unroll
    for (int w = 0; w < U::kWords; ++w) {
      float x[8];
      load8(row + (g + 4 * i) * U::kChannels + 8 * w, wide, x);
      bf16x8 terms[kFp4Terms<T>];
      fp4_terms(x, terms);
#pragma unroll
      for (int p = 0; p < kFp4Terms<T>; ++p) qf[p][i * U::kWords + w] = terms[p];
    }
}

// Scores of 16 keys from `key` on that the column does not see become minus infinity; the bits of those it sees.  (The bits first, then a score at a time
// by its bit: sixteen comparisons kept as they are spill 63 to 85 scalar registers.)
__device__ __forceinline__ uint32_t mask_scores(f32x4 (&sc)[4], int key, bool known, int from, int pos, int end) {
  const int first = min(max(from - key, 0), 16), last = known ? min(max(min(pos, end - 1) - key + 1, first), 16) : first;
  const uint32_t seen = (1u << last) - (1u << first);
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const uint32_t in = (uint32_t)__builtin_amdgcn_sbfe((int)seen, 4 * j + x, 1);   // all bits or none
      sc[j][x] = __uint_as_float((__float_as_uint(sc[j][x]) & in) | (0xff800000u & ~in));
    }
  return seen;
}

// One step of the running softmax of a column (this lane's 16 keys of 64, of which it sees `seen`): probabilities as the product's operand, sums rescaled
// where the maximum grows.  The maximum is that of the scores as they are, and what is scaled is their difference: a scaled maximum is rounded, by 2^-4 at
// 2^20 and 2^32 at 2^56, which the probabilities of a tile share, but not those of the next one.  (One operation a score more than scores scaled by the
// multiplication that subtracts: 2,048 rows of 32 heads of 128 73.5 us for 72.2.)  Their sum is a product with ones, of what the values are multiplied by
// and over all 64 (added up by the lanes: 64 requests of 4,096 keys 123 us for 122, the prompt 74.0 for 73.7).  PT terms a probability.
template <int PT, int NB>
__device__ __forceinline__ void soften(const f32x4 (&sc)[4], uint32_t seen, float scale, float& m, f32x4& l, f32x4 (&o)[2 * NB], bf16x8 (&pf)[PT][2]) {
  float top = seen ? -kLargest : -__builtin_inff();
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int x = 0; x < 4; ++x) top = fmaxf(top, sc[j][x]);
  const float now = fmaxf(m, quads_max(top));   // (the scale is positive)
  if (__any(now > m)) {
    const float shrink = now > m ? __builtin_amdgcn_exp2f((m - now) * scale) : 1.f;
    m = now;
    l[0] *= shrink;
#pragma unroll
    for (int b = 0; b < 2 * NB; ++b)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[b][x] *= shrink;
  }
  const float least = m == -__builtin_inff() ? 0.f : m;
  float p[16];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int x = 0; x < 4; ++x) p[4 * j + x] = __builtin_amdgcn_exp2f((sc[j][x] - least) * scale);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = p[8 * c + e];
    bf16x8 terms[PT];
    fp4_terms(x, terms);
#pragma unroll
    for (int q = 0; q < PT; ++q) {
      pf[q][c] = terms[q];
      l = mfma(bf16x8{} + (bf16)1.f, terms[q], l);
    }
  }
}

// Eight tokens of a byte row of values: the operands of channels i (low) and i + 16.
__device__ __forceinline__ void values8(uint32_t w0, uint32_t w1, uint32_t s0, uint32_t s1, bf16x8& low, bf16x8& high) {
  uint32_t two[8];   // both channels of a token
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t w = e < 4 ? w0 : w1;
    const float unit = fp4_unit_of(e < 4 ? s0 : s1, e % 4);
    bf16x2 y;
    if (e % 4 == 0) y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 0);
    else if (e % 4 == 1) y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 1);
    else if (e % 4 == 2) y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 2);
    else y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 3);
    two[e] = __builtin_bit_cast(uint32_t, y);
  }
  u32x4 a, b;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    a[e] = __builtin_amdgcn_perm(two[2 * e + 1], two[2 * e], 0x05040100u);
    b[e] = __builtin_amdgcn_perm(two[2 * e + 1], two[2 * e], 0x07060302u);
  }
  low = __builtin_bit_cast(bf16x8, a);
  high = __builtin_bit_cast(bf16x8, b);
}

// A probability of zero times a value that is not finite is not zero: the blocks that are marked so take part as finite ones, and are
// counted for the columns that see them, which become NaN.  Scales and seen keys of eight tokens.
__device__ __forceinline__ void count_bad(uint32_t s0, uint32_t s1, uint32_t seen, f32x4& count) {
  bf16x8 is, sees;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    is[e] = ((e < 4 ? s0 : s1) >> (8 * (e % 4)) & 255u) == kFp4BadScale ? (bf16)1.f : (bf16)0.f;
    sees[e] = seen >> e & 1u ? (bf16)1.f : (bf16)0.f;
  }
  count = mfma(is, sees, count);
}

// 0xff in each byte of a word of four tokens from `key` on that some column sees
__device__ __forceinline__ uint32_t kept_bytes(int key, int from, int to) {
  uint32_t keep = 0;
#pragma unroll
  for (int x = 0; x < 4; ++x) keep |= key + x >= from && key + x < to ? 0xffu << (8 * x) : 0u;
  return keep;
}

// a tile of 64 keys and values as a lane takes them from memory
template <int NB> struct Tile {
  uint32_t kw[4][NB], ks[Units<NB>::kCount];
  u32x4 vw[NB], vs[NB];
};
template <int NB> __device__ __forceinline__ void load_tile(const AttendArgs& a, const Places& at, int kvh, int r, int g, Tile<NB>& t) {
  using U = Units<NB>;
  const size_t block = fp4_block_bytes(a.page), head_bytes = block * NB;
  const uint8_t* kb = a.k + page_at(a, at.kp, kvh, head_bytes);
  const uint8_t* vb = a.v + page_at(a, at.vp, kvh, head_bytes);
  const int kslot = r & 3;
#pragma unroll
  for (int i = 0; i < U::kCount; ++i) {
    const int u = g + 4 * i;
    const uint8_t* base = kb + (size_t)(u * U::kChannels / kFp4Block) * block;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      __builtin_memcpy(&t.kw[j][i * U::kWords], __builtin_assume_aligned(base + (at.koff + 4 * j + kslot) * 16 + u * U::kChannels % kFp4Block / 2, 4 * U::kWords),
                       4 * U::kWords);
    t.ks[i] = *reinterpret_cast<const uint32_t*>(base + 16 * a.page + at.koff + 4 * kslot);
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    t.vw[b] = *reinterpret_cast<const u32x4*>(vb + (size_t)b * block + (size_t)r * a.page + at.voff);
    t.vs[b] = *reinterpret_cast<const u32x4*>(vb + (size_t)b * block + (size_t)16 * a.page + at.voff);
  }
}

// R tiles of 16 columns over a tile of keys: their scores, the step of their softmax, their sums.  first, last: the columns' positions;
// [lo, end): keys that some column may see.
template <typename T, int NB, int R> struct Columns {
  static constexpr int SP = kFp4Terms<T>, PT = SP > 1 ? SP : 2;
  bf16x8 qf[R][SP][NB];
  f32x4 o[R][2 * NB];
  float m[R];
  f32x4 l[R];   // (the first of four is the sum)
  int pos[R], from[R];   // a column sees the keys from .. pos

  __device__ __forceinline__ void begin(const AttendArgs& a, int q_start, int pos0, int kvh, int c0, int cols, int r, int g) {
#pragma unroll
    for (int t = 0; t < R; ++t) {
      const int c = min(c0 + 16 * t + r, cols - 1);
      pos[t] = pos0 + c / a.rep;
      from[t] = window_from(a, pos[t]);
      load_query<T, NB>((const T*)a.q + (size_t)(q_start + c / a.rep) * a.q_stride + (size_t)(kvh * a.rep + c % a.rep) * (NB * kFp4Block), g, a.q_wide, qf[t]);
      m[t] = -__builtin_inff();
      l[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < 2 * NB; ++b) o[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  __device__ __forceinline__ void take(const AttendArgs& a, Tile<NB>& w, int t0, bool known, int first, int last, int lo, int end, int g) {
    const int key = t0 + 16 * g;   // this lane's 16
    f32x4 sc[R][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int t = 0; t < R; ++t) sc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const bf16x8 kf = fp4_unpack8(w.kw[j][i], fp4_unit_of(w.ks[i / Units<NB>::kWords], j));
#pragma unroll
        for (int t = 0; t < R; ++t)
#pragma unroll
          for (int p = 0; p < SP; ++p) sc[t][j] = mfma(kf, qf[t][p][i], sc[t][j]);
      }
    }
    // tiles that some column sees in part
    const bool whole = t0 + kTile <= first + 1 && t0 + kTile <= end && (a.window <= 0 || t0 > last - a.window) && __all(known);
    bool bad = false;   // a value that may be behind a mask stands in a block that is not finite
    uint32_t seen[R];
#pragma unroll
    for (int t = 0; t < R; ++t) seen[t] = 0xffffu;
    if (!whole) {
#pragma unroll
      for (int t = 0; t < R; ++t) seen[t] = mask_scores(sc[t], key, known, from[t], pos[t], end);
      // (what no column sees, the rest of a last page among it, may be anything: its scales become the smallest)
      uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t keep = known ? kept_bytes(key + 4 * e, lo, end) : 0u;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          w.vs[b][e] &= keep;
          any |= bytes_255(w.vs[b][e]);
        }
      }
      bad = __any(any != 0);
    }
    bf16x8 pf[R][PT][2];
#pragma unroll
    for (int t = 0; t < R; ++t) soften<PT, NB>(sc[t], seen[t], a.scale, m[t], l[t], o[t], pf[t]);
    if (__builtin_expect(bad, 0)) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int t = 0; t < R; ++t) {
          f32x4 count = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 2; ++c) count_bad(w.vs[b][2 * c], w.vs[b][2 * c + 1], seen[t] >> (8 * c), count);
          if (count[0] > 0.f) o[t][2 * b] = o[t][2 * b + 1] = f32x4{} + __builtin_nanf("");
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) w.vs[b][e] &= ~bytes_255(w.vs[b][e]);   // 255 becomes 127
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        bf16x8 low, high;
        values8(w.vw[b][2 * c], w.vw[b][2 * c + 1], w.vs[b][2 * c], w.vs[b][2 * c + 1], low, high);
#pragma unroll
        for (int p = 0; p < PT; ++p)
#pragma unroll
          for (int t = 0; t < R; ++t) {
            o[t][2 * b] = mfma(low, pf[t][p][c], o[t][2 * b]);
            o[t][2 * b + 1] = mfma(high, pf[t][p][c], o[t][2 * b + 1]);
          }
      }
  }
};

// Waves a SIMD holds at least: what just fits the registers.  (Without the bound a few more registers cost a wave: 64 requests of 4,096 keys, 32 heads of
// 64, 124 us, with it 122; 2,048 rows of 32 heads of 128 110 and 74.)
template <typename T, int NB, int R> constexpr int least_waves = NB > 4 ? 1 : std::is_same_v<T, float> || R > 1 ? 2 : NB > 2 ? 3 : 4;

// Few columns: the waves of a workgroup share out the tiles of keys.  T the rows' type, NB blocks a head, W waves.  Bound by memory: 64 requests of
// 4,096 keys, 32 heads of 64, 119 to 125 us for 571 MB (4.7 TB/s); 64 of 4,000, 8 kv heads of 128, 61 us (4.6 TB/s).
template <typename T, int NB, int W>
__global__ __launch_bounds__(W * kWave) __attribute__((amdgpu_waves_per_eu(least_waves<T, NB, 1>))) void fp4_attend_keys_kernel(AttendArgs a) {
  constexpr int D = NB * kFp4Block;
  const int lane = threadIdx.x % kWave, r = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int id = blockIdx.x;
  const int kvh = id % a.nkv;
  id /= a.nkv;
  const int c0 = id % a.col_tiles * 16;
  id /= a.col_tiles;
  const int split = id % a.splits, s = id / a.splits;

  const int q_start = a.q_start[s], pos0 = min(a.pos0[s], INT32_MAX - a.max_q);
  const int cols = q_start < 0 ? 0 : min(min(a.q_len[s], a.max_q), a.n - q_start) * a.rep;
  if (c0 >= cols) return;   // (the whole workgroup)
  const int first = pos0 + c0 / a.rep, last = pos0 + min(cols - 1, c0 + 15) / a.rep;   // positions of the columns
  const int limit = max(0, min(last + 1, a.table_cols * a.page)), lo = min(window_from(a, first), limit);
  const int begin = (int)min((long long)(lo & ~(kTile - 1)) + (long long)split * a.chunk, (long long)limit), end = begin + min(limit - begin, a.chunk);

  // the numbers of a tile's pages are asked for a tile ahead, those of the first before the queries
  const int32_t* table = a.tables + (size_t)s * a.table_stride;
  const int start = begin + wave * kTile;
  Places at = look_up(a, table, start + 16 * (r >> 2), start + 16 * g);
  Columns<T, NB, 1> columns;
  columns.begin(a, q_start, pos0, kvh, c0, cols, r, g);
  for (int t0 = start; t0 < end; t0 += W * kTile) {
    const bool known = known_page(a, at.vp);
    Tile<NB> tile;
    load_tile(a, at, kvh, r, g, tile);
    at = look_up(a, table, t0 + W * kTile + 16 * (r >> 2), t0 + W * kTile + 16 * g);
    columns.take(a, tile, t0, known, first, last, lo, end, g);
  }

  constexpr int kPad = 4, kThreads = W * 4, kEach = D / kThreads;   // threads a column, channels a thread
  __shared__ float so[W][16][D + kPad];
  __shared__ float sm[W][16], sl[W][16];
  if (g == 0) sm[wave][r] = columns.m[0], sl[wave][r] = columns.l[0][0];
#pragma unroll
  for (int b = 0; b < 2 * NB; ++b) *reinterpret_cast<f32x4*>(&so[wave][r][16 * b + 4 * g]) = columns.o[0][b];
  __syncthreads();
  const int column = threadIdx.x / kThreads, part = threadIdx.x % kThreads, c = c0 + column;
  if (c >= cols) return;
  float top = sm[0][column], sum = 0.f, weight[W];
#pragma unroll
  for (int w = 1; w < W; ++w) top = fmaxf(top, sm[w][column]);
#pragma unroll
  for (int w = 0; w < W; ++w) {
    weight[w] = sm[w][column] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((sm[w][column] - top) * a.scale);
    sum += weight[w] * sl[w][column];
  }
  float x[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    x[e] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) x[e] = fmaf(weight[w], so[w][column][part * kEach + e], x[e]);
  }
  if (a.splits > 1) {
    const size_t to = (((size_t)s * a.nkv + kvh) * a.max_q * a.rep + c) * a.splits + split;
    if (part == 0) a.ml[to] = make_float2(top, sum);
#pragma unroll
    for (int e = 0; e < kEach; ++e) a.acc[to * D + part * kEach + e] = x[e];
  } else {
    const float over = over_sum(sum, top);
    T* row = (T*)a.out + (size_t)(q_start + c / a.rep) * a.out_stride + (size_t)(kvh * a.rep + c % a.rep) * D;
#pragma unroll
    for (int e = 0; e < kEach; ++e) row[part * kEach + e] = (T)(x[e] * over);
  }
}

// More columns: each of four waves has R tiles of its own and takes all keys.  Bound by the conversions, the softmax and the products, which add up: 2,048
// rows of 32 heads of 128 in 73 us (the same rows over a bf16 cache in the prefill kernel: 56).  A request's long tiles of columns come first and its
// short ones behind them in turn, so that compute units of two workgroups have about the same to do: in their order 94.  Making a tile bf16 once for
// the four waves, through LDS, took half as long again (95 for 64, with probabilities of one term): the barriers cost more than the conversions that they save.
template <typename T, int NB, int R>
__global__ __launch_bounds__(4 * kWave) __attribute__((amdgpu_waves_per_eu(least_waves<T, NB, R>))) void fp4_attend_cols_kernel(AttendArgs a) {
  constexpr int D = NB * kFp4Block, C = 16 * R;
  const int lane = threadIdx.x % kWave, r = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // kv heads fastest: the workgroups of one request and kv head, which read the same keys, are a multiple of nkv apart and, where
  // that is a multiple of 8, on one XCD
  int id = blockIdx.x;
  const int kvh = id % a.nkv;
  id /= a.nkv;
  const int turn = id % a.col_tiles, col_tile = turn < a.col_tiles / 2 ? a.col_tiles - 1 - turn : turn - a.col_tiles / 2;
  id /= a.col_tiles;
  const int split = id % a.splits, s = id / a.splits;

  const int q_start = a.q_start[s], pos0 = min(a.pos0[s], INT32_MAX - a.max_q);
  const int cols = q_start < 0 ? 0 : min(min(a.q_len[s], a.max_q), a.n - q_start) * a.rep;
  const int c0 = (col_tile * 4 + wave) * C;
  if (c0 >= cols) return;   // (the wave: there is no barrier)
  const int first = pos0 + c0 / a.rep, last = pos0 + min(cols - 1, c0 + C - 1) / a.rep;   // positions of the wave's columns
  const int limit = max(0, min(last + 1, a.table_cols * a.page)), lo = min(window_from(a, first), limit);
  const int begin = (int)min((long long)(lo & ~(kTile - 1)) + (long long)split * a.chunk, (long long)limit), end = begin + min(limit - begin, a.chunk);

  const int32_t* table = a.tables + (size_t)s * a.table_stride;
  Places at = look_up(a, table, begin + 16 * (r >> 2), begin + 16 * g);
  Columns<T, NB, R> columns;
  columns.begin(a, q_start, pos0, kvh, c0, cols, r, g);
  for (int t0 = begin; t0 < end; t0 += kTile) {
    const bool known = known_page(a, at.vp);
    Tile<NB> tile;
    load_tile(a, at, kvh, r, g, tile);
    at = look_up(a, table, t0 + kTile + 16 * (r >> 2), t0 + kTile + 16 * g);
    columns.take(a, tile, t0, known, first, last, lo, end, g);
  }

#pragma unroll
  for (int t = 0; t < R; ++t) {
    const float sum = columns.l[t][0];
    const int c = c0 + 16 * t + r;
    if (c >= cols) continue;
    if (a.splits > 1) {
      const size_t to = (((size_t)s * a.nkv + kvh) * a.max_q * a.rep + c) * a.splits + split;
      if (g == 0) a.ml[to] = make_float2(columns.m[t], sum);
#pragma unroll
      for (int b = 0; b < 2 * NB; ++b) *reinterpret_cast<f32x4*>(a.acc + to * D + 16 * b + 4 * g) = columns.o[t][b];
    } else {
      const float over = over_sum(sum, columns.m[t]);
      T* row = (T*)a.out + (size_t)(q_start + c / a.rep) * a.out_stride + (size_t)(kvh * a.rep + c % a.rep) * D;
#pragma unroll
      for (int b = 0; b < 2 * NB; ++b) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = columns.o[t][b][e] * over;
        store4<T>(row + 16 * b + 4 * g, a.out_wide, x);
      }
    }
  }
}

// Joins the runs of a context: a wave a column, lane i the weight of run i.
template <typename T, int D>
__global__ __launch_bounds__(256) void fp4_join_kernel(AttendArgs a, int columns) {
  const int lane = threadIdx.x % kWave, at = blockIdx.x * 4 + threadIdx.x / kWave;
  if (at >= columns) return;
  const int per = a.max_q * a.rep, c = at % per, kvh = at / per % a.nkv, s = at / per / a.nkv;
  const int q_start = a.q_start[s], token = c / a.rep;
  if (q_start < 0 || token >= min(a.q_len[s], a.n - q_start)) return;
  const float2 ml = lane < a.splits ? a.ml[(size_t)at * a.splits + lane] : make_float2(-__builtin_inff(), 0.f);
  const float top = wave_max(ml.x);
  const float weight = ml.x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((ml.x - top) * a.scale);
  const float sum = wave_sum(weight * ml.y), over = over_sum(sum, top);
  constexpr int kEach = (D + kWave - 1) / kWave;
  float x[kEach] = {};
  // (runs in which a column sees nothing have left zeros; what is read again behind the last has no weight)
  for (int i = 0; i < a.splits; i += 8) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float w = __shfl(weight, i + k, kWave);
      const float* run = a.acc + ((size_t)at * a.splits + min(i + k, a.splits - 1)) * D;
#pragma unroll
      for (int e = 0; e < kEach; ++e) x[e] = fmaf(w, run[min(lane + e * kWave, D - 1)], x[e]);
    }
  }
  T* row = (T*)a.out + (size_t)(q_start + token) * a.out_stride + (size_t)(kvh * a.rep + c % a.rep) * D;
#pragma unroll
  for (int e = 0; e < kEach; ++e)
    if (lane + e * kWave < D) row[lane + e * kWave] = (T)(x[e] * over);
}

struct Plan {
  bool cols;
  int r, col_tiles, splits, chunk;
};

// How a launch is laid out: a function of its sizes and the rows' type alone.
static Plan plan(int n_seqs, int nkv, int rep, int hd, int max_q, int max_context, int window, int dtype) {
  const long long columns = (long long)max_q * rep;
  auto laid_out = [&](bool cols, int r, long long runs, long long least, long long grain) {
    const int width = cols ? 64 * r : 16;   // columns a workgroup
    const long long tokens = std::min<long long>(max_q, (16 * r - 1) / rep + 2);   // of a wave's columns
    const long long span = window > 0 ? std::min<long long>(max_context, window + tokens + kTile) : max_context;
    const long long chunk = std::min<long long>(std::max(least, ((span + runs - 1) / runs + grain - 1) / grain * grain), 1 << 30);
    return Plan{cols, r, (int)((columns + width - 1) / width), (int)std::max<long long>(1, (span + chunk - 1) / chunk), (int)chunk};
  };
  // Few columns, runs of a context: as many workgroups as compute units have one, none of fewer than 512 keys; 129 to 217 workgroups of long contexts
  // in three.  Over 110 sizes 1.6 % slower than the best number of runs.  us: one request of 4,000 keys and 32 kv heads in 8 runs 9.2, in 4 10.7;
  // 256 workgroups in one run 19.4, in two 22.1; 160 (5 of 9,000) in three 29.2, in two 37.6.  More than 256 stay whole: 40 requests of 1,000 to 8,000 keys
  // and 8 kv heads 62.2, in three 61.8, though 10 of 9,000 and 32 kv heads take 60.6 and 49.1.
  if (columns <= 32) {
    const long long groups = (long long)n_seqs * nkv * ((columns + 15) / 16);
    long long runs = std::max<long long>(1, std::min<long long>(256 / groups, kMostSplits));
    if (groups > 128 && groups < 218 && max_context >= 4096) runs = 3;
    if (max_context <= 1024) runs = 1;
    return laid_out(false, 1, runs, 512, 8 * kTile);
  }
  // More: one tile of columns a wave, two (where they fit the registers) or three (heads of 64: of 32 they gain nothing), and as many runs, as take least by a model with numbers fitted to some 3,000
  // launches (154 sizes: its choice is 1.5 % slower than the best, at most 19): a wave's turns, each `alone` us; the tiles that a SIMD has to do on
  // average, `busy` us each, more where the workgroups do not divide evenly by the compute units; the joining of runs, its launch and its
  // bytes.  us: 131 rows behind 3,900, 32 heads of 64 and as many kv heads, three tiles in 8 runs 27.0, in 16 27.4, two in 11 27.7, one in 11 29.6; 8 kv
  // heads of 128 two in 6 35.5, in 8 44.3, one in 11 38.2; 1,024 rows of 32 heads of 64 one in one run 19.7, two 27.1; 2,048 rows of 32 heads of 64 two in one
  // 53, one 59; 8 x 50 rows behind 550 one in one 20.3, two in two 27.8; 131 rows behind 15,869, 32 heads of 64, three in 16 64.8, two 75.8, one 77.3.
  static constexpr float kAlone[3][9] = {{0.f, 0.38f, 0.48f, 1.2f, 0.75f, 0.f, 0.f, 0.f, 1.f}, {0.f, 0.61f, 0.65f, 1.49f, 1.11f}, {0.f, 0.f, 1.2f}};   // by tiles and blocks a head
  static constexpr float kBusy[3][9] = {{0.f, 0.57f, 0.72f, 1.21f, 0.92f, 0.f, 0.f, 0.f, 2.42f}, {0.f, 0.89f, 1.2f, 1.8f, 1.36f}, {0.f, 0.f, 1.08f}};
  const bool wide = dtype == kF32;
  Plan best{};
  float least = 0.f;
  for (int r = 1; r <= (wide || hd > 128 ? 1 : hd == 64 ? 3 : 2); ++r) {
    const float alone = kAlone[r - 1][hd / 32] * (wide ? 1.4f : 1.f), busy = kBusy[r - 1][hd / 32] * (wide ? 1.4f : 1.f);
    const float waves = (float)n_seqs * nkv * (float)((columns + 16 * r - 1) / (16 * r));
    for (int runs : {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 28, 32, 40, 48, 64}) {
      const Plan p = laid_out(true, r, runs, kTile, kTile);
      const float groups = (float)n_seqs * nkv * p.col_tiles * p.splits / 256, span = std::min((float)max_context, (float)p.chunk * p.splits);
      if (runs > 1 && groups > 32) break;
      const float seen = window > 0 ? span : std::max(span - max_q / 2.f, span / 2);   // keys of a row, on average
      float us = p.chunk / 64.f * alone + waves * seen / 64 / 1024 * busy * (1 + 0.6f * (std::ceil(groups) / groups - 1));
      if (p.splits > 1) us += 2.5f + (float)n_seqs * max_q * nkv * rep * (hd + 2) * p.splits / 500e3f;
      if (best.splits == 0 || us < least) least = us, best = p;
    }
  }
  return best;
}

template <typename T, int NB> static void launch(const Plan& p, const AttendArgs& a, int n_seqs, hipStream_t stream) {
  constexpr int W = NB == 8 ? 4 : 8;   // (the waves' sums of heads of 256 would not fit LDS twice)
  const dim3 grid((unsigned)((long long)n_seqs * a.nkv * p.col_tiles * p.splits));
  if (!p.cols) hipLaunchKernelGGL((fp4_attend_keys_kernel<T, NB, W>), grid, dim3(W * kWave), 0, stream, a);
  else if (p.r == 1) hipLaunchKernelGGL((fp4_attend_cols_kernel<T, NB, 1>), grid, dim3(4 * kWave), 0, stream, a);
  else if constexpr (std::is_same_v<T, bf16> && NB <= 4) {
    if (p.r == 2) hipLaunchKernelGGL((fp4_attend_cols_kernel<T, NB, 2>), grid, dim3(4 * kWave), 0, stream, a);
    else if constexpr (NB == 2) hipLaunchKernelGGL((fp4_attend_cols_kernel<T, NB, 3>), grid, dim3(4 * kWave), 0, stream, a);
  }
  if (p.splits > 1) {
    const int columns = n_seqs * a.nkv * a.max_q * a.rep;
    hipLaunchKernelGGL((fp4_join_kernel<T, NB * kFp4Block>), dim3((columns + 3) / 4), dim3(256), 0, stream, a, columns);
  }
}

}  // namespace gb

using namespace gb;

static bool takes(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 256; }

// floats of workspace; 0: none is needed
extern "C" long long gb_fp4_attention_floats(int n_seqs, int nh, int nkv, int hd, int max_q, int max_context, int window, int dtype) {
  if (!takes(hd) || n_seqs <= 0 || nkv <= 0 || nh < nkv || max_q <= 0 || max_context <= 0) return 0;
  const Plan p = plan(n_seqs, nkv, nh / nkv, hd, max_q, max_context, window, dtype);
  return p.splits > 1 ? (long long)n_seqs * nh * max_q * p.splits * (hd + 2) : 0;
}

extern "C" int gb_fp4_attention(const void* q, int q_stride, void* out, int out_stride, int dtype, int n, const int32_t* q_start,
                                const int32_t* q_len, const int32_t* pos0, int n_seqs, int max_q, int max_context, const int32_t* tables,
                                int table_stride, int table_cols, const void* k_pages, const void* v_pages, int pages, int nh, int nkv, int hd,
                                int page, float scale, int window, float* workspace, long long workspace_floats, hipStream_t stream) {
  GB_REQUIRE(takes(hd), "fp4_attention: heads of %d channels: 32, 64, 96, 128 or 256", hd);
  GB_REQUIRE(n >= 0 && n_seqs >= 0 && nkv > 0 && nh > 0 && nh % nkv == 0, "fp4_attention: bad sizes n=%d requests=%d heads=%d/%d", n, n_seqs, nh, nkv);
  GB_REQUIRE(page > 0 && page % 16 == 0 && pages > 0 && table_cols > 0, "fp4_attention: pages of %d slots, %d pages, %d table columns", page, pages,
             table_cols);
  GB_REQUIRE((long long)nh * hd <= q_stride && (long long)nh * hd <= out_stride, "fp4_attention: row strides %d, %d are shorter than the heads", q_stride,
             out_stride);
  GB_REQUIRE(dtype == kF32 || dtype == kBF16, "fp4_attention: unknown dtype %d", dtype);
  GB_REQUIRE(max_q >= 0 && max_context >= 0 && (long long)table_cols * page <= INT32_MAX - 1024, "fp4_attention: rows %d, context %d, tables of %d pages", max_q,
             max_context, table_cols);
  if (n == 0 || n_seqs == 0 || max_q == 0) return 0;
  const int rep = nh / nkv;
  const Plan p = plan(n_seqs, nkv, rep, hd, max_q, std::max(1, max_context), window, dtype);
  const long long columns = (long long)n_seqs * nh * max_q, groups = (long long)n_seqs * nkv * p.col_tiles * p.splits;
  // (a last workgroup's columns, up to 192 and most of them none of the request's, have numbers of 32 bits too)
  GB_REQUIRE(columns <= INT32_MAX - 1024 && groups < (1ll << 31), "fp4_attention: too many rows for one launch");
  const long long need = p.splits > 1 ? columns * p.splits * (hd + 2) : 0;
  GB_REQUIRE(need == 0 || (workspace && workspace_floats >= need), "fp4_attention: a workspace of %lld floats is needed, %lld are given", need,
             workspace ? workspace_floats : 0ll);
  const int e = dtype == kF32 ? 4 : 2;
  AttendArgs a{};
  a.q = q, a.out = out, a.q_start = q_start, a.q_len = q_len, a.pos0 = pos0, a.tables = tables;
  a.k = (const uint8_t*)k_pages, a.v = (const uint8_t*)v_pages;
  a.acc = workspace, a.ml = reinterpret_cast<float2*>(workspace + columns * p.splits * hd);
  a.q_stride = q_stride, a.out_stride = out_stride, a.n = n, a.table_stride = table_stride, a.table_cols = table_cols, a.pages = pages;
  a.nkv = nkv, a.rep = rep, a.page = page, a.page_shift = (page & (page - 1)) == 0 ? __builtin_ctz(page) : -1, a.max_q = max_q;
  a.window = window, a.chunk = p.chunk, a.splits = p.splits, a.col_tiles = p.col_tiles;
  a.scale = scale * 1.44269504088896340736f;
  a.q_wide = ((uintptr_t)q & 15) == 0 && (size_t)q_stride * e % 16 == 0;
  a.out_wide = ((uintptr_t)out & 15) == 0 && (size_t)out_stride * e % 16 == 0;
#define GB_FP4_LAUNCH(NB)                                                   \
  case NB * kFp4Block:                                                      \
    if (dtype == kF32) launch<float, NB>(p, a, n_seqs, stream);             \
    else launch<bf16, NB>(p, a, n_seqs, stream);                            \
    break;
  switch (hd) {
    GB_FP4_LAUNCH(1) GB_FP4_LAUNCH(2) GB_FP4_LAUNCH(3) GB_FP4_LAUNCH(4) GB_FP4_LAUNCH(8)
  }
  return launched("fp4_attention");
}

GB_TAPED(gb_fp4_attention)
GB_DEFINE_LAST_ERROR
