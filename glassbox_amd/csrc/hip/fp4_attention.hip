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
// A row of 32 bits counts as three bf16 terms (fp4.h), and so do its probabilities; a bf16 row's probabilities are rounded to bf16, as
// its result is.
//
// Few columns (decoding): the waves of a workgroup share out the tiles and are joined through LDS; a long context is cut into runs
// for several workgroups, joined by a second kernel.  More columns: each wave has columns of its own and all of a run's keys.
#include "fp4.h"

#include <algorithm>

namespace gb {

constexpr int kTile = 64;        // keys a wave takes at a time
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
__device__ __forceinline__ float quads_sum(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t w = __float_as_uint(__uint_as_float(a[0]) + __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
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

// T the rows' type, NB blocks a head, R column tiles a wave, W waves, COLS: the waves have columns of their own.  (Two waves a SIMD at least
// where they do: without the bound 2,048 rows of 32 heads of 128 take 108 us, with it 84.)
template <typename T, int NB, int R, int W, bool COLS>
__global__ __launch_bounds__(W * kWave) __attribute__((amdgpu_waves_per_eu(COLS && NB <= 4 ? 2 : 1))) void fp4_attend_kernel(AttendArgs a) {
  using U = Units<NB>;
  constexpr int D = NB * kFp4Block, SP = kFp4Terms<T>, C = 16 * R;
  static_assert(COLS || R == 1, "waves that share their columns hold one tile of them");
  const int lane = threadIdx.x % kWave, r = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // kv heads fastest: the workgroups of one request and kv head, which read the same keys, are a multiple of nkv apart and, where
  // that is a multiple of 8, on one XCD
  int id = blockIdx.x;
  const int kvh = id % a.nkv;
  id /= a.nkv;
  const int col_tile = id % a.col_tiles;
  id /= a.col_tiles;
  const int split = id % a.splits, s = id / a.splits;

  const int q_start = a.q_start[s], pos0 = a.pos0[s];
  const int q_len = min(min(a.q_len[s], a.max_q), a.n - q_start);
  const int cols = q_start < 0 ? 0 : q_len * a.rep;
  const int c0 = (col_tile * (COLS ? W : 1) + (COLS ? wave : 0)) * C;
  if (c0 >= cols) return;   // (without COLS the whole workgroup)
  const int first = pos0 + c0 / a.rep, last = pos0 + min(cols - 1, c0 + C - 1) / a.rep;   // positions of this wave's columns
  const int lo = a.window > 0 ? max(0, first - a.window + 1) : 0;
  const int begin = (lo & ~(kTile - 1)) + split * a.chunk;
  const int end = min(min(last + 1, a.table_cols * a.page), begin + a.chunk);

  // The numbers of a tile's pages are asked for a tile ahead, those of the first before the queries.  What is no page of the pool is not
  // read (page 0 is, in its place), its keys are not seen.
  const int32_t* table = a.tables + (size_t)s * a.table_stride;
  const int start = begin + (COLS ? 0 : wave * kTile), stride = COLS ? kTile : W * kTile;
  int kp, vp, koff, voff;   // of this lane's keys, 16 tokens all of which one page holds, and of its values
  auto look_up = [&](int t0) {
    const int kt = t0 + 16 * (r >> 2), vt = t0 + 16 * g;
    const int ki = a.page_shift >= 0 ? kt >> a.page_shift : kt / a.page, vi = a.page_shift >= 0 ? vt >> a.page_shift : vt / a.page;
    koff = kt - ki * a.page;
    voff = vt - vi * a.page;
    const int k0 = table[min(ki, a.table_cols - 1)], v0 = table[min(vi, a.table_cols - 1)];
    kp = ki < a.table_cols ? k0 : -1;
    vp = vi < a.table_cols ? v0 : -1;
  };
  look_up(start);

  int pos[R], from[R];   // a column sees the keys from .. pos
  bool own[R];
  bf16x8 qf[R][SP][NB];
#pragma unroll
  for (int t = 0; t < R; ++t) {
    const int c = c0 + 16 * t + r;
    own[t] = c < cols;
    const int cc = own[t] ? c : cols - 1;
    pos[t] = pos0 + cc / a.rep;
    from[t] = a.window > 0 ? pos[t] - a.window + 1 : 0;
    const T* row = (const T*)a.q + (size_t)(q_start + cc / a.rep) * a.q_stride + (size_t)(kvh * a.rep + cc % a.rep) * D;
#pragma unroll
    for (int i = 0; i < U::kCount; ++i)
#pragma unroll
      for (int w = 0; w < U::kWords; ++w) {
        float x[8];
        load8(row + (g + 4 * i) * U::kChannels + 8 * w, a.q_wide, x);
        bf16x8 terms[SP];
        fp4_terms(x, terms);
#pragma unroll
        for (int p = 0; p < SP; ++p) qf[t][p][i * U::kWords + w] = terms[p];
      }
  }

  f32x4 o[R][2 * NB];
  float m[R], l[R];
#pragma unroll
  for (int t = 0; t < R; ++t) {
    m[t] = -__builtin_inff();
    l[t] = 0.f;
#pragma unroll
    for (int b = 0; b < 2 * NB; ++b) o[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const size_t block = fp4_block_bytes(a.page), head_bytes = block * NB;
  const int kslot = r & 3;
  for (int t0 = start; t0 < end; t0 += stride) {
    const int vt = t0 + 16 * g;
    const bool known = (unsigned)vp < (unsigned)a.pages;
    const uint8_t* kb = a.k + ((size_t)((unsigned)kp < (unsigned)a.pages ? kp : 0) * a.nkv + kvh) * head_bytes;
    const uint8_t* vb = a.v + ((size_t)(known ? vp : 0) * a.nkv + kvh) * head_bytes;

    uint32_t kw[4][NB], ks[U::kCount];
    u32x4 vw[NB], vs[NB];
#pragma unroll
    for (int i = 0; i < U::kCount; ++i) {
      const int u = g + 4 * i, b = u * U::kChannels / kFp4Block, in = u * U::kChannels % kFp4Block / 2;
      const uint8_t* base = kb + (size_t)b * block;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint8_t* p = base + (koff + 4 * j + kslot) * 16 + in;
        if constexpr (U::kWords == 4) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
          for (int e = 0; e < 4; ++e) kw[j][4 * i + e] = w[e];
        } else if constexpr (U::kWords == 2) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(p);
          kw[j][2 * i] = w[0], kw[j][2 * i + 1] = w[1];
        } else {
          kw[j][i] = *reinterpret_cast<const uint32_t*>(p);
        }
      }
      ks[i] = *reinterpret_cast<const uint32_t*>(base + 16 * a.page + koff + 4 * kslot);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      vw[b] = *reinterpret_cast<const u32x4*>(vb + (size_t)b * block + (size_t)r * a.page + voff);
      vs[b] = *reinterpret_cast<const u32x4*>(vb + (size_t)b * block + (size_t)16 * a.page + voff);
    }
    look_up(t0 + stride);

    f32x4 sc[R][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int t = 0; t < R; ++t) sc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < U::kCount; ++i)
#pragma unroll
        for (int w = 0; w < U::kWords; ++w) {
          const bf16x8 kf = fp4_unpack8(kw[j][i * U::kWords + w], fp4_unit(ks[i] >> (8 * j) & 255u));
#pragma unroll
          for (int t = 0; t < R; ++t)
#pragma unroll
            for (int p = 0; p < SP; ++p) sc[t][j] = mfma(kf, qf[t][p][i * U::kWords + w], sc[t][j]);
        }
    }

    // tiles that some column sees in part
    const bool whole = t0 + kTile <= first + 1 && t0 + kTile <= end && (a.window <= 0 || t0 > last - a.window) && __all(known);
    bool bad = false;      // a value of this tile that may be behind a mask stands in a block that is not finite
    uint32_t seen[R];      // of this lane's 16 keys
#pragma unroll
    for (int t = 0; t < R; ++t) seen[t] = 0xffffu;
    if (!whole) {
#pragma unroll
      for (int t = 0; t < R; ++t) {
        seen[t] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int key = vt + 4 * j + x;
            const bool in = known && key <= pos[t] && key >= from[t] && key < end;
            seen[t] |= in ? 1u << (4 * j + x) : 0u;
            sc[t][j][x] = in ? sc[t][j][x] : -__builtin_inff();
          }
      }
      // (what no column sees, the rest of a last page among it, may be anything: its scales become the smallest)
      uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t keep = 0;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int key = vt + 4 * e + x;
          keep |= known && key >= lo && key <= last && key < end ? 0xffu << (8 * x) : 0u;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          vs[b][e] &= keep;
          any |= bytes_255(vs[b][e]);
        }
      }
      bad = __any(any != 0);
    }

    bf16x8 pf[R][SP][2];
#pragma unroll
    for (int t = 0; t < R; ++t) {
      float top = -__builtin_inff();
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) top = fmaxf(top, sc[t][j][x]);
      // scale is positive or the maximum is of the scaled scores: see below
      top = quads_max(top) * a.scale;
      const float now = fmaxf(m[t], top);
      if (__any(now > m[t])) {
        const float shrink = now > m[t] ? __builtin_amdgcn_exp2f(m[t] - now) : 1.f;
        m[t] = now;
        l[t] *= shrink;
#pragma unroll
        for (int b = 0; b < 2 * NB; ++b)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[t][b][x] *= shrink;
      }
      const float sub = m[t] == -__builtin_inff() ? 0.f : m[t];
      float p[16], sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          p[4 * j + x] = __builtin_amdgcn_exp2f(fmaf(sc[t][j][x], a.scale, -sub));
          sum += p[4 * j + x];
        }
      l[t] += sum;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = p[8 * c + e];
        bf16x8 terms[SP];
        fp4_terms(x, terms);
#pragma unroll
        for (int q = 0; q < SP; ++q) pf[t][q][c] = terms[q];
      }
    }

    if (__builtin_expect(bad, 0)) {
      // a probability of zero times a value that is not finite is not zero: such blocks are counted for the columns that see
      // them, which become NaN, and take part as finite ones
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        f32x4 count[R];
#pragma unroll
        for (int t = 0; t < R; ++t) count[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          bf16x8 is;
#pragma unroll
          for (int e = 0; e < 8; ++e) is[e] = (vs[b][2 * c + e / 4] >> (8 * (e % 4)) & 255u) == kFp4BadScale ? (bf16)1.f : (bf16)0.f;
#pragma unroll
          for (int t = 0; t < R; ++t) {
            bf16x8 sees;
#pragma unroll
            for (int e = 0; e < 8; ++e) sees[e] = seen[t] >> (8 * c + e) & 1u ? (bf16)1.f : (bf16)0.f;
            count[t] = mfma(is, sees, count[t]);
          }
        }
#pragma unroll
        for (int t = 0; t < R; ++t)
          if (count[t][0] > 0.f) o[t][2 * b] = o[t][2 * b + 1] = f32x4{} + __builtin_nanf("");
#pragma unroll
        for (int e = 0; e < 4; ++e) vs[b][e] &= ~bytes_255(vs[b][e]);   // 255 becomes 127
      }
    }

#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t two[8];   // channels r (low) and r + 16 of a token
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float unit = fp4_unit(vs[b][2 * c + e / 4] >> (8 * (e % 4)) & 255u);
          const uint32_t w = vw[b][2 * c + e / 4];
          bf16x2 y;
          if (e % 4 == 0) y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 0);
          else if (e % 4 == 1) y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 1);
          else if (e % 4 == 2) y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 2);
          else y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, 3);
          two[e] = __builtin_bit_cast(uint32_t, y);
        }
        u32x4 low, high;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          low[e] = __builtin_amdgcn_perm(two[2 * e + 1], two[2 * e], 0x05040100u);
          high[e] = __builtin_amdgcn_perm(two[2 * e + 1], two[2 * e], 0x07060302u);
        }
        const bf16x8 vl = __builtin_bit_cast(bf16x8, low), vh = __builtin_bit_cast(bf16x8, high);
#pragma unroll
        for (int t = 0; t < R; ++t)
#pragma unroll
          for (int p = 0; p < SP; ++p) {
            o[t][2 * b] = mfma(vl, pf[t][p][c], o[t][2 * b]);
            o[t][2 * b + 1] = mfma(vh, pf[t][p][c], o[t][2 * b + 1]);
          }
      }
  }
#pragma unroll
  for (int t = 0; t < R; ++t) l[t] = quads_sum(l[t]);

  const size_t column0 = ((size_t)s * a.nkv + kvh) * a.max_q * a.rep;   // of the partial results
  if constexpr (COLS) {
#pragma unroll
    for (int t = 0; t < R; ++t) {
      if (!own[t]) continue;
      const int c = c0 + 16 * t + r;
      if (a.splits > 1) {
        const size_t at = (column0 + c) * a.splits + split;
        if (g == 0) a.ml[at] = make_float2(m[t], l[t]);
#pragma unroll
        for (int b = 0; b < 2 * NB; ++b) *reinterpret_cast<f32x4*>(a.acc + at * D + 16 * b + 4 * g) = o[t][b];
      } else {
        const float over = l[t] > 0.f || l[t] != l[t] ? 1.f / l[t] : 0.f;
        T* row = (T*)a.out + (size_t)(q_start + c / a.rep) * a.out_stride + (size_t)(kvh * a.rep + c % a.rep) * D;
#pragma unroll
        for (int b = 0; b < 2 * NB; ++b) {
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = o[t][b][e] * over;
          store4<T>(row + 16 * b + 4 * g, a.out_wide, x);
        }
      }
    }
  } else {
    constexpr int kPad = 4, kThreads = W * 4, kEach = D / kThreads;   // threads a column, channels a thread
    __shared__ float so[W][16][D + kPad];
    __shared__ float sm[W][16], sl[W][16];
    if (g == 0) sm[wave][r] = m[0], sl[wave][r] = l[0];
#pragma unroll
    for (int b = 0; b < 2 * NB; ++b) *reinterpret_cast<f32x4*>(&so[wave][r][16 * b + 4 * g]) = o[0][b];
    __syncthreads();
    const int column = threadIdx.x / kThreads, part = threadIdx.x % kThreads, c = c0 + column;
    if (c >= cols) return;
    float top = sm[0][column], sum = 0.f, weight[W];
#pragma unroll
    for (int w = 1; w < W; ++w) top = fmaxf(top, sm[w][column]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      weight[w] = sm[w][column] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(sm[w][column] - top);
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
      const size_t at = (column0 + c) * a.splits + split;
      if (part == 0) a.ml[at] = make_float2(top, sum);
#pragma unroll
      for (int e = 0; e < kEach; ++e) a.acc[at * D + part * kEach + e] = x[e];
    } else {
      const float over = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
      T* row = (T*)a.out + (size_t)(q_start + c / a.rep) * a.out_stride + (size_t)(kvh * a.rep + c % a.rep) * D;
#pragma unroll
      for (int e = 0; e < kEach; ++e) row[part * kEach + e] = (T)(x[e] * over);
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
  const float weight = ml.x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ml.x - top);
  const float sum = wave_sum(weight * ml.y), over = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  constexpr int kEach = (D + kWave - 1) / kWave;
  float x[kEach] = {};
  // (runs in which a column sees nothing have left zeros)
#pragma unroll 8
  for (int i = 0; i < a.splits; ++i) {
    const float w = __shfl(weight, i, kWave);
#pragma unroll
    for (int e = 0; e < kEach; ++e) x[e] = fmaf(w, a.acc[((size_t)at * a.splits + i) * D + min(lane + e * kWave, D - 1)], x[e]);
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
  Plan p;
  const long long columns = (long long)max_q * rep;
  p.cols = columns > 32;
  // Waves with columns of their own: two tiles of them where there are many and they fit the registers (2,048 rows of 32 heads of 128: 84 us,
  // one tile 96; 120 rows of 5 requests, 3 heads a kv head: 7.7 and 5.9; 64 rows behind 8,000, 4 a kv head: 37.7 and 36.5).
  p.r = p.cols && columns >= 1024 && dtype == kBF16 && hd <= 128 ? 2 : 1;
  const int width = p.cols ? 64 * p.r : 16;
  p.col_tiles = (int)((columns + width - 1) / width);
  const long long tokens = std::min<long long>(max_q, (16 * p.r - 1) / rep + 2);
  const long long span = window > 0 ? std::min<long long>(max_context, window + tokens + kTile) : max_context;
  // Runs of a context: about as many workgroups as compute units (half as many again of four waves), none of fewer than 1,024 keys (256).  us:
  // 4 requests of 16,000 keys and 8 kv heads in 8 runs 23.6, in 4 29.6, in 16 28.7; 256 workgroups in one run 18.2, in two 21.9; 131 rows behind
  // 3,900, 32 heads, in 8 30, in 4 34.
  const long long groups = (long long)n_seqs * nkv * p.col_tiles;
  const long long want = ((p.cols ? 512 : 256) + groups / 2) / groups, least = p.cols ? 256 : 1024, grain = p.cols ? kTile : 8 * kTile;
  const long long runs = std::max<long long>(1, std::min<long long>(want, kMostSplits));
  const long long chunk = std::max(least, ((span + runs - 1) / runs + grain - 1) / grain * grain);
  p.splits = (int)std::max<long long>(1, (span + chunk - 1) / chunk);
  p.chunk = (int)chunk;
  return p;
}

template <typename T, int NB> static void launch(const Plan& p, const AttendArgs& a, int n_seqs, hipStream_t stream) {
  constexpr int W = NB == 8 ? 4 : 8;   // (the waves' sums of heads of 256 would not fit LDS twice)
  const dim3 grid((unsigned)((long long)n_seqs * a.nkv * p.col_tiles * p.splits));
  if (!p.cols) hipLaunchKernelGGL((fp4_attend_kernel<T, NB, 1, W, false>), grid, dim3(W * kWave), 0, stream, a);
  else if (p.r == 1) hipLaunchKernelGGL((fp4_attend_kernel<T, NB, 1, 4, true>), grid, dim3(4 * kWave), 0, stream, a);
  else if constexpr (std::is_same_v<T, bf16> && NB <= 4) hipLaunchKernelGGL((fp4_attend_kernel<T, NB, 2, 4, true>), grid, dim3(4 * kWave), 0, stream, a);
  if (p.splits > 1) {
    const int columns = n_seqs * a.nkv * a.max_q * a.rep;
    hipLaunchKernelGGL((fp4_join_kernel<T, NB * kFp4Block>), dim3((columns + 3) / 4), dim3(256), 0, stream, a, columns);
  }
}

}  // namespace gb

using namespace gb;

extern "C" int gb_fp4_attention_takes(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 256; }

// floats of workspace; 0: none is needed
extern "C" long long gb_fp4_attention_floats(int n_seqs, int nh, int nkv, int hd, int max_q, int max_context, int window, int dtype) {
  if (n_seqs <= 0 || nkv <= 0 || nh < nkv || max_q <= 0 || max_context <= 0) return 0;
  const Plan p = plan(n_seqs, nkv, nh / nkv, hd, max_q, max_context, window, dtype);
  return p.splits > 1 ? (long long)n_seqs * nh * max_q * p.splits * (hd + 2) : 0;
}

extern "C" int gb_fp4_attention(const void* q, int q_stride, void* out, int out_stride, int dtype, int n, const int32_t* q_start,
                                const int32_t* q_len, const int32_t* pos0, int n_seqs, int max_q, int max_context, const int32_t* tables,
                                int table_stride, int table_cols, const void* k_pages, const void* v_pages, int pages, int nh, int nkv, int hd,
                                int page, float scale, int window, float* workspace, long long workspace_floats, hipStream_t stream) {
  GB_REQUIRE(gb_fp4_attention_takes(hd), "fp4_attention: heads of %d channels: 32, 64, 96, 128 or 256", hd);
  GB_REQUIRE(n >= 0 && n_seqs >= 0 && nkv > 0 && nh > 0 && nh % nkv == 0, "fp4_attention: bad sizes n=%d requests=%d heads=%d/%d", n, n_seqs, nh, nkv);
  GB_REQUIRE(page > 0 && page % 16 == 0 && pages > 0 && table_cols > 0, "fp4_attention: pages of %d slots, %d pages, %d table columns", page, pages,
             table_cols);
  GB_REQUIRE((long long)nh * hd <= q_stride && (long long)nh * hd <= out_stride, "fp4_attention: row strides %d, %d are shorter than the heads", q_stride,
             out_stride);
  GB_REQUIRE(dtype == kF32 || dtype == kBF16, "fp4_attention: unknown dtype %d", dtype);
  GB_REQUIRE(max_q >= 0 && max_context >= 0 && (long long)table_cols * page < (1ll << 31), "fp4_attention: rows %d, context %d, tables of %d pages", max_q,
             max_context, table_cols);
  if (n == 0 || n_seqs == 0 || max_q == 0) return 0;
  const int rep = nh / nkv;
  const Plan p = plan(n_seqs, nkv, rep, hd, max_q, std::max(1, max_context), window, dtype);
  const long long columns = (long long)n_seqs * nh * max_q, groups = (long long)n_seqs * nkv * p.col_tiles * p.splits;
  GB_REQUIRE(columns < (1ll << 31) && groups < (1ll << 31), "fp4_attention: too many rows for one launch");
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
