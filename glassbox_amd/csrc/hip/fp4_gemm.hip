// Products with four-bit weights (fp4.h): out (+)= a . W^T, or silu(a . gate^T) * (a . up^T) of a stack of both.
//
// W is the left operand of 16 x 16 x 32 products: a lane holds 32 neighbours of one row of W, a block: 16 bytes and a scale, which become
// bf16 in registers, two numbers an instruction, exactly, and never see LDS.  32-bit rows count as three bf16 terms (fp4.h): the
// products stay exact; all sums are in 32 bits.  Workgroups too few for the chip divide k into slices, which a second kernel adds up in
// order (given a workspace).  Two kernels:
//
// lines (few rows): bound by W's bytes, 17 / 32 of one a number, and from a few rows on by what a compute unit brings in of a.  8 rows
//   of W a tile, lanes r >= 8 with the same rows 128 numbers further on, so that a wave's load reads 8 whole lines of 128 bytes; the rows of
//   a stand in the columns likewise, 8 of them, and of the 16 x 16 results the two quarters in which both are of one run of k are added up.
//   The waves of a workgroup take turns over k and are joined through LDS.  (16 rows of W and half lines, us: 1 row by 128,256 of 4,096
//   68.5, whole lines 62: 4.5 TB/s; 28,672 of 4,096 20.3 and 19; 2,048 of 8,192 7.1 and 5.4.)
// tiles (more): a's rows go through LDS, 64 or 32 of them by 64 to 256 rows of W, whose waves have rows of W of their own: 2,048 rows by
//   28,672 of 4,096 in 537 us, 0.9 PFLOP/s; 64 rows in 39.  (Rows of a from memory to every wave: 60; what bounds it there is the way into a
//   compute unit, 20 to 50 GB/s each.)
// Measured and left: workgroups that go on from tile to tile with the next one's lines under way (8 rows by 28,672 of 4,096 25.6, like this 21.6:
// more registers, fewer waves); an RMS norm of the rows on the way (41, and 25.5 with the norm in a launch of its own: rows of 32 bits and
// gamma are three times the bytes into every compute unit).  What a norm costs up to 8 rows, where the product before prepares it (gamma x in bf16 and
// partial sums of squares) and this one divides by the root: 8 rows by 4,096 of 4,096, then by 28,672 27.6 us for both, 29.6 with a launch between.
#include "fp4.h"

#include <algorithm>
#include <cmath>

namespace gb {

struct GemmArgs {
  const void* x;
  const uint8_t *codes, *scales;
  void* out;
  float* slices;   // [slices, M, N]: given, each slice of k leaves its sums there
  // Of RMS norms, up to 8 bf16 rows.  parts: the rows are bf16(gamma x) of an x whose squares' sums these are, [n_parts, 8], to be added up; h: the
  // product adds into such an x, and writes bf16(gamma x) there and a tile's sums of squares to sums [n_tiles, 8].
  const float* parts;
  const void* gamma;
  bf16* h;
  float* sums;
  int n_parts, gamma32, ldh;
  float eps;
  int ldx, ldo, M, N, blocks, scale_stride, n_tiles, m_tiles, turns, epilogue, out32, out_wide;   // epilogue 0 store, 1 add, 2 silu(gate) * up
};

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// four neighbouring columns of a row of out, those below `limit`
__device__ __forceinline__ void put(const GemmArgs& a, int m, int n, int limit, f32x4 v) {
  const size_t at = (size_t)m * a.ldo + n;
  if (a.out32) {
    float* o = (float*)a.out + at;
    if (a.out_wide && n + 4 <= limit) {
      if (a.epilogue == 1) v += *reinterpret_cast<const f32x4*>(o);
      *reinterpret_cast<f32x4*>(o) = v;
      return;
    }
    for (int i = 0; i < 4 && n + i < limit; ++i) o[i] = a.epilogue == 1 ? o[i] + v[i] : v[i];
  } else {
    bf16* o = (bf16*)a.out + at;
    if (a.out_wide && n + 4 <= limit) {
      *reinterpret_cast<bf16x4*>(o) = bf16x4{(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
      return;
    }
    for (int i = 0; i < 4 && n + i < limit; ++i) o[i] = (bf16)v[i];
  }
}

// the same, or into the slice of k whose sum it is
__device__ __forceinline__ void put_or_leave(const GemmArgs& a, int m, int n, int limit, f32x4 v) {
  if (!a.slices) return put(a, m, n, limit, v);
  float* o = a.slices + ((size_t)blockIdx.y * a.M + m) * a.N + n;
  if ((a.N | n) % 4 == 0 && n + 4 <= limit) *reinterpret_cast<f32x4*>(o) = v;   // (an up half may begin anywhere)
  else
    for (int i = 0; i < 4 && n + i < limit; ++i) o[i] = v[i];
}

// eight elements of a row as they come from memory
template <typename T> struct Raw {
  u32x4 w[std::is_same_v<T, float> ? 2 : 1];
};
template <typename T> __device__ __forceinline__ void keep(Raw<T>& v, bool in) {   // zeros where not
#pragma unroll
  for (auto& w : v.w)
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = in ? w[e] : 0u;
}
__device__ __forceinline__ void terms_of(const Raw<bf16>& v, bf16x8 (&out)[1]) { out[0] = __builtin_bit_cast(bf16x8, v.w[0]); }
__device__ __forceinline__ void terms_of(const Raw<float>& v, bf16x8 (&out)[3]) {
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(v.w[e / 4][e % 4]);
  fp4_terms(x, out);
}

// T the rows' type, MT tiles of 8 rows of a, NT of 8 rows of W (with silu every other one of the up half), W waves, U blocks of 32 numbers of
// k that a lane asks for at once; NORMS: takes part in norms (GemmArgs)
template <typename T, int MT, int NT, int W, int U, bool NORMS>
__global__ __launch_bounds__(W * kWave) __attribute__((amdgpu_waves_per_eu(MT * NT * kFp4Terms<T> == 16 ? 2 : 1))) void fp4_lines_kernel(GemmArgs a) {
  constexpr int SP = kFp4Terms<T>;
  const int lane = threadIdx.x % kWave, r = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // the row tiles of one tile of W follow each other on one XCD (workgroups go to the eight in turn), whose L2 then has it
  const int order = blockIdx.x / 8, nt = order / a.m_tiles * 8 + blockIdx.x % 8, mt0 = order % a.m_tiles * 8 * MT;
  if (nt >= a.n_tiles) return;
  const bool silu = a.epilogue == 2;
  const int half = a.N / 2;
  const uint8_t *codes[NT], *scales[NT];
  const T* x[MT];
  auto row_of = [&](int p) { return silu ? (p & 1 ? half : 0) + (nt * (NT / 2) + p / 2) * 8 : (nt * NT + p) * 8; };
#pragma unroll
  for (int p = 0; p < NT; ++p) {
    const int row = min(row_of(p) + r % 8, (silu && !(p & 1) ? half : a.N) - 1);
    codes[p] = a.codes + (size_t)row * a.blocks * 16;
    scales[p] = a.scales + (size_t)row * a.scale_stride;
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) x[t] = (const T*)a.x + (size_t)min(mt0 + t * 8 + r % 8, a.M - 1) * a.ldx;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int p = 0; p < NT; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[p][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  // this lane's u-th block in turn i.  Loads do not branch: beyond the end they read the last block again
  auto block = [&](int i, int u) { return 8 * ((i * W + wave) * U + u) + 4 * (r / 8) + g; };
  u32x4 next[U][NT];
  uint32_t next_scale[U][NT];
  Raw<T> next_x[U][MT][4];
  auto fetch = [&](int i) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = min(block(i, u), a.blocks - 1);
#pragma unroll
      for (int p = 0; p < NT; ++p) {
        next[u][p] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(codes[p] + (size_t)c * 16));
        next_scale[u][p] = scales[p][c];
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int w = 0; w < 4; ++w)   // (rows may begin anywhere: the hardware takes 16 bytes from any address)
          __builtin_memcpy(&next_x[u][t][w], x[t] + (size_t)c * kFp4Block + 8 * w, sizeof(Raw<T>));
    }
  };
  const int first = blockIdx.y * a.turns, turns = (a.blocks - 8 * U * wave + 8 * U * W - 1) / (8 * U * W), end = min(turns, first + a.turns);   // this wave's
  // (the last turn stands by itself: a load behind a branch would be waited for together with all others)
  auto turn = [&](int i, auto last) {
    u32x4 now[U][NT];
    float unit[U][NT];
    Raw<T> raw[U][MT][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = !last || block(i, u) < a.blocks;   // what is beyond the end counts as zero
#pragma unroll
      for (int p = 0; p < NT; ++p) now[u][p] = next[u][p], unit[u][p] = in ? fp4_unit(next_scale[u][p]) : 0.f;
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          raw[u][t][w] = next_x[u][t][w];
          if constexpr (last) keep(raw[u][t][w], in);
        }
    }
    if constexpr (!last) fetch(i + 1);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        bf16x8 xf[MT][SP];
#pragma unroll
        for (int t = 0; t < MT; ++t) terms_of(raw[u][t][w], xf[t]);
#pragma unroll
        for (int p = 0; p < NT; ++p) {
          const bf16x8 kf = fp4_unpack8(now[u][p][w], unit[u][p]);
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int q = 0; q < SP; ++q) acc[p][t] = mfma(kf, xf[t][q], acc[p][t]);
        }
      }
  };
  static_assert(!NORMS || (MT == 1 && std::is_same_v<T, bf16>), "norms are of up to 8 bf16 rows");
  // partial sums of four rows, which are added up behind the products; a word in turn, the rows' halves in turn.  (a.sums: of no meaning)
  constexpr int kWords = 8 / W;   // a thread: 256 parts
  f32x4 some[kWords];
  if (first < end) fetch(first);
  if constexpr (NORMS)
#pragma unroll
    for (int k = 0; k < kWords; ++k)
      some[k] = *reinterpret_cast<const f32x4*>((a.parts ? a.parts : a.sums) + 4 * min((int)threadIdx.x + k * W * kWave, max(2 * a.n_parts - 1, 0)));
  if (first < end) {
    for (int i = first; i + 1 < end; ++i) turn(i, std::false_type{});
    turn(end - 1, std::true_type{});
  }

  __shared__ f32x4 part[W][NT * MT][kWave];
  __shared__ float wave_sums[W][8], tile_sums[NT][8];
  if constexpr (NORMS) {
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kWords; ++k)
      if ((int)threadIdx.x + k * W * kWave < 2 * a.n_parts) sum += some[k];
    for (int i = threadIdx.x + kWords * W * kWave; i < 2 * a.n_parts; i += W * kWave) sum += *reinterpret_cast<const f32x4*>(a.parts + 4 * (size_t)i);
#pragma unroll
    for (int d = 2; d < kWave; d *= 2)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], d);
    if (lane < 2) *reinterpret_cast<f32x4*>(&wave_sums[wave][4 * lane]) = sum;
  }
#pragma unroll
  for (int p = 0; p < NT; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t) part[wave][p * MT + t][lane] = acc[p][t];
  __syncthreads();
  float root = 1.f;
  if constexpr (NORMS) {
    if (a.parts) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) sum += wave_sums[w][r % 8];
      root = 1.f / sqrtf(sum / (a.blocks * kFp4Block) + a.eps);
    }
  }
  // lane (r, g) of a tile's total: rows 4 g .. of W, row r of a; the quarters g < 2, r < 8 and g >= 2, r >= 8 are of two runs of k
  auto total = [&](int tile) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) v += part[w][tile][lane] + part[w][tile][lane ^ 40];
    if constexpr (NORMS) v *= root;
    return v;
  };
  if (silu && !a.slices) {
    for (int u = wave; u < NT / 2 * MT; u += W) {
      const int p = u / MT * 2, t = u % MT, m = mt0 + 8 * t + r;
      const f32x4 gate = total(p * MT + t), up = total((p + 1) * MT + t);
      f32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = silu_times(gate[i], up[i]);
      if (m < a.M && r < 8 && g < 2) put(a, m, row_of(p) + 4 * g, half, v);
    }
  } else if (NORMS && a.h) {
    for (int p = wave; p < NT; p += W) {
      const f32x4 v = total(p);
      const int n = row_of(p) + 4 * g;
      float squares = 0.f;
      if (r < a.M && r < 8 && g < 2 && n < a.N) {
        f32x4* o = reinterpret_cast<f32x4*>((float*)a.out + (size_t)r * a.ldo + n);
        const f32x4 x = *o + v;
        *o = x;
        bf16x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float gamma = a.gamma32 ? ((const float*)a.gamma)[n + i] : (float)((const bf16*)a.gamma)[n + i];
          y[i] = (bf16)(gamma * x[i]);
          squares = fmaf(x[i], x[i], squares);
        }
        *reinterpret_cast<bf16x4*>(a.h + (size_t)r * a.ldh + n) = y;
      }
      squares += __shfl_xor(squares, 16);
      if (lane < 8) tile_sums[p][lane] = squares;
    }
    __syncthreads();
    if (threadIdx.x < 8) {
      float sum = 0.f;
#pragma unroll
      for (int p = 0; p < NT; ++p) sum += tile_sums[p][threadIdx.x];
      a.sums[(size_t)nt * 8 + threadIdx.x] = sum;
    }
  } else {
    for (int u = wave; u < NT * MT; u += W) {
      const int p = u / MT, t = u % MT, m = mt0 + 8 * t + r;
      const f32x4 v = total(u);
      if (m < a.M && r < 8 && g < 2) put_or_leave(a, m, row_of(p) + 4 * g, silu && !(p & 1) ? half : a.N, v);
    }
  }
}

// T the rows' type, MT tiles of 16 rows of a (all waves'), NT of 16 rows of W a wave, B blocks of 32 numbers of k a step.  a's rows pass
// through LDS, a step ahead in registers, the words of a row exchanged by the row so that the operands' reads spread over the banks.
template <typename T, int MT, int NT, int B>
__global__ __launch_bounds__(256) void fp4_tiles_kernel(GemmArgs a) {
  constexpr int SP = kFp4Terms<T>, W = 4, U = B / 4, kRows = 16 * MT, kWords = 4 * B, kLoads = kRows * kWords / 256, kStep = 256 / kWords;
  __shared__ bf16x8 xs[2][SP][kRows * kWords];
  const int lane = threadIdx.x % kWave, r = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int order = blockIdx.x / 8, nt = order / a.m_tiles * 8 + blockIdx.x % 8, mt0 = order % a.m_tiles * kRows;   // (as above)
  if (nt >= a.n_tiles) return;
  const bool silu = a.epilogue == 2;
  const int half = a.N / 2;
  const uint8_t *codes[NT], *scales[NT];
  auto row_of = [&](int p) {
    const int i = (nt * W + wave) * NT + p;
    return silu ? (i & 1 ? half : 0) + i / 2 * 16 : i * 16;
  };
#pragma unroll
  for (int p = 0; p < NT; ++p) {
    const int row = min(row_of(p) + r, (silu && !(p & 1) ? half : a.N) - 1);
    codes[p] = a.codes + (size_t)row * a.blocks * 16;
    scales[p] = a.scales + (size_t)row * a.scale_stride;
  }
  const int word = threadIdx.x % kWords, row0 = threadIdx.x / kWords;   // what this thread brings of a: eight numbers of every kStep-th row
  const T* x[kLoads];
#pragma unroll
  for (int l = 0; l < kLoads; ++l) x[l] = (const T*)a.x + (size_t)min(mt0 + row0 + l * kStep, a.M - 1) * a.ldx;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int p = 0; p < NT; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[p][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  u32x4 next[U][NT];
  uint32_t next_scale[U][NT];
  Raw<T> next_x[kLoads];
  auto fetch = [&](int i) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = min(i * B + U * g + u, a.blocks - 1);
#pragma unroll
      for (int p = 0; p < NT; ++p) {
        next[u][p] = *reinterpret_cast<const u32x4*>(codes[p] + (size_t)c * 16);
        next_scale[u][p] = scales[p][c];
      }
    }
    const int c = min(i * B + word / 4, a.blocks - 1);
#pragma unroll
    for (int l = 0; l < kLoads; ++l) __builtin_memcpy(&next_x[l], x[l] + (size_t)c * kFp4Block + word % 4 * 8, sizeof(Raw<T>));
  };
  auto bring = [&](int i, int buffer) {
    const bool in = i * B + word / 4 < a.blocks;
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      const int row = row0 + l * kStep;
      Raw<T> v = next_x[l];
      keep(v, in);
      bf16x8 terms[SP];
      terms_of(v, terms);
#pragma unroll
      for (int q = 0; q < SP; ++q) xs[buffer][q][row * kWords + (word ^ (row & 15))] = terms[q];
    }
  };
  const int first = blockIdx.y * a.turns, turns = (a.blocks + B - 1) / B, end = min(turns, first + a.turns);
  auto turn = [&](int i, int buffer, auto last) {
    u32x4 now[U][NT];
    float unit[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = i * B + U * g + u < a.blocks;
#pragma unroll
      for (int p = 0; p < NT; ++p) now[u][p] = next[u][p], unit[u][p] = in ? fp4_unit(next_scale[u][p]) : 0.f;
    }
    if constexpr (!last) fetch(i + 1);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        bf16x8 kf[NT];
#pragma unroll
        for (int p = 0; p < NT; ++p) kf[p] = fp4_unpack8(now[u][p][w], unit[u][p]);
#pragma unroll
        for (int q = 0; q < SP; ++q) {
          bf16x8 xf[MT];
#pragma unroll
          for (int t = 0; t < MT; ++t) xf[t] = xs[buffer][q][(16 * t + r) * kWords + (((U * g + u) * 4 + w) ^ r)];
#pragma unroll
          for (int p = 0; p < NT; ++p)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[p][t] = mfma(kf[p], xf[t], acc[p][t]);
        }
      }
    if constexpr (!last) {   // into the half that was read a turn ago: every wave has passed the barrier behind that
      bring(i + 1, buffer ^ 1);
      __syncthreads();
    }
  };
  fetch(first);
  bring(first, 0);
  __syncthreads();
  int buffer = 0;
  for (int i = first; i + 1 < end; ++i, buffer ^= 1) turn(i, buffer, std::false_type{});
  turn(end - 1, buffer, std::true_type{});

  // lane (r, g): row r of a tile of a, rows 4 g .. of W
#pragma unroll
  for (int p = 0; p < NT; ++p) {
    const int n = row_of(p) + 4 * g;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int m = mt0 + 16 * t + r;
      if (m >= a.M) continue;
      if (!silu || a.slices) {
        put_or_leave(a, m, n, silu && !(p & 1) ? half : a.N, acc[p][t]);
      } else if (p & 1) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = silu_times(acc[p - 1][t][e], acc[p][t][e]);
        put(a, m, n - half, half, v);
      }
    }
  }
}

// Adds up the slices of k, in their order, and does what the epilogue does.  A thread a column (of both halves, with silu).
__global__ __launch_bounds__(256) void fp4_gemm_join_kernel(GemmArgs a, int slices) {
  const int cols = a.epilogue == 2 ? a.N / 2 : a.N;
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  const int m = (int)(at / cols), n = (int)(at % cols);
  if (m >= a.M) return;
  const size_t step = (size_t)a.M * a.N;
  const float* p = a.slices + (size_t)m * a.N + n;
  float v = 0.f, u = 0.f;
#pragma unroll 8
  for (int z = 0; z < slices; ++z) {
    v += p[z * step];
    if (a.epilogue == 2) u += p[z * step + cols];
  }
  if (a.epilogue == 2) v = silu_times(v, u);
  const size_t o = (size_t)m * a.ldo + n;
  if (!a.out32) ((bf16*)a.out)[o] = (bf16)v;
  else if (a.epilogue == 1) ((float*)a.out)[o] += v;
  else ((float*)a.out)[o] = v;
}

// The same for a product that adds to the residual, a workgroup a row; with the new row in hand it does the RMS norm that reads it next as well:
// h = bf16(gamma (x s)), s = 1 / sqrt(mean(x^2) + eps).  A thread has up to two words of four columns, whose slices it asks for eight at a time.  Bound by
// the way into the few compute units that have a row.  us with the product, and with the norm in a launch of its own: 16 rows by 2,048 of 8,192 10.2 and 11.7, 64
// 12.8 and 14.9, 512 33.0 and 36.5; 40 by 4,096 of 14,336 25.0 and 26.6, by 4,096 of 4,096 13.4 and 15.1.
constexpr int kNormColumns = 2 * 4 * 1024;
__global__ __launch_bounds__(1024) void fp4_gemm_join_norm_kernel(GemmArgs a, int slices) {
  __shared__ float partial[16];
  const int m = blockIdx.x, threads = blockDim.x;
  const size_t step = (size_t)a.M * a.N;
  f32x4 x[2];
  float gamma[2][4], squares = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int n = 4 * ((int)threadIdx.x + i * threads);
    if (n >= a.N) break;
    const float* p = a.slices + (size_t)m * a.N + n;
    f32x4* o = reinterpret_cast<f32x4*>((float*)a.out + (size_t)m * a.ldo + n);
    const f32x4 old = *o;
#pragma unroll
    for (int e = 0; e < 4; ++e) gamma[i][e] = a.gamma32 ? ((const float*)a.gamma)[n + e] : (float)((const bf16*)a.gamma)[n + e];
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int z = 0; z < slices; z += 8) {
      f32x4 v[8];   // (behind the last slice the last again, not added)
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const f32x4*>(p + min(z + k, slices - 1) * step);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (z + k < slices) sum += v[k];
    }
    x[i] = old + sum;
    *o = x[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) squares = fmaf(x[i][e], x[i][e], squares);
  }
  squares = wave_sum(squares);
  if (threadIdx.x % kWave == 0) partial[threadIdx.x / kWave] = squares;
  __syncthreads();
  float total = 0.f;
  for (int w = 0; w < threads / kWave; ++w) total += partial[w];
  const float s = 1.f / sqrtf(total / a.N + a.eps);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int n = 4 * ((int)threadIdx.x + i * threads);
    if (n >= a.N) break;
    bf16x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (bf16)(gamma[i][e] * (x[i][e] * s));
    *reinterpret_cast<bf16x4*>(a.h + (size_t)m * a.ldh + n) = y;
  }
}

// Which kernel takes a product, and how: a function of its sizes and type alone.
struct Form {
  int rows_w, rows_a, step;          // a workgroup's rows of W and of a, blocks of k a turn
  float alone[2], busy[2];           // us of a turn with little and with much on the chip (bf16 rows, 32-bit ones), 0: not for such rows
};
static constexpr int kLinesForms = 7;
static constexpr int kNormRows = 8;   // up to which a product takes part in norms (lines, with k whole)
static constexpr Form kForms[] = {{32, 8, 64, {0.f, 0.f}, {1.9f, 3.1f}},         // lines: MT x NT 1 x 4, 8 waves
                                  {16, 8, 64, {0.f, 0.f}, {1.35f, 2.3f}},        // 1 x 2, 8
                                  {8, 8, 128, {0.f, 0.f}, {1.7f, 3.7f}},         // 1 x 1, 8 (U 2)
                                  {64, 16, 32, {0.f, 0.f}, {2.3f, 4.9f}},        // 2 x 8, 4
                                  {32, 16, 64, {0.f, 0.f}, {2.9f, 5.5f}},        // 2 x 4, 8
                                  {32, 8, 32, {0.f, 0.f}, {0.f, 0.f}},           // 1 x 4, 4 (not beyond 8 rows)
                                  {64, 8, 32, {0.f, 0.f}, {0.f, 0.f}},           // 1 x 8, 4 (nor this)
                                  {64, 32, 8, {0.95f, 0.f}, {0.6f, 0.f}},        // tiles: 2 x 1, 8 blocks
                                  {128, 32, 8, {1.4f, 0.f}, {1.05f, 0.f}},       // 2 x 2, 8
                                  {128, 64, 8, {2.f, 0.f}, {1.4f, 0.f}},         // 4 x 2, 8
                                  {256, 64, 4, {1.65f, 0.f}, {1.05f, 0.f}},      // 4 x 4, 4
                                  {64, 32, 4, {0.f, 1.2f}, {0.f, 0.67f}},        // 2 x 1, 4
                                  {128, 32, 4, {0.f, 1.35f}, {0.f, 0.87f}}};     // 2 x 2, 4
struct Plan {
  int form, n_tiles, m_tiles, turns, slices;
};

static Plan plan(int M, int N, int K, bool silu, int dtype, int most_slices) {
  auto laid_out = [&](int form, int slices) {
    const Form& f = kForms[form];
    Plan p{form, silu ? (N / 2 + f.rows_w / 2 - 1) / (f.rows_w / 2) : (N + f.rows_w - 1) / f.rows_w, (M + f.rows_a - 1) / f.rows_a, 0, 0};
    const int turns = (K / 32 + f.step - 1) / f.step;
    p.turns = (turns + slices - 1) / slices;
    p.slices = (turns + p.turns - 1) / p.turns;
    return p;
  };
  // up to 8 rows: as many rows of W a workgroup as leave about 192 of them (16 with silu, which takes pairs of tiles).  us, 8 rows: 6,144 of
  // 4,096 by 32 7.8, by 16 8.5; 2,560 of 2,560 by 16 5.3, by 8 6.1; 2,048 of 8,192 by 8 8.1, by 16 11.
  // Many rows of W: workgroups of four waves, which take more turns each: 1 row by 128,256 of 4,096 62, in eight waves 66; by 49,152 of 2,048 13.7 and
  // 16.8.  With more rows of a, and 32-bit ones, by 64 rows of W: 4 rows by 128,256 of 4,096 61, by 32 69, in eight waves 70 (by 49,152 of 2,048
  // 16.8, 15.8, 18.3); 8 by 28,672 of 4,096 21.6, by 32 24.0, in eight waves 24.2; 8 32-bit ones 27.8 and, in eight waves, 35.3.  k has no part in the
  // choice: whoever takes a norm's partial sums asks for their number without it.
  if (M <= kNormRows) {
    if (N >= 16384 && M <= (N < 24576 ? 4 : 2) && dtype == kBF16) return laid_out(5, 1);
    if (N >= 24576 || (N >= 16384 && M > 4)) return laid_out(6, 1);
    return laid_out(N >= 6144 ? 0 : N >= 2560 || silu ? 1 : 2, 1);
  }
  // more: the form with the least time by a model, whose numbers are fitted to 21 products of 9 to 1,024 rows in every form, with weights from
  // memory (8 % off; its choice is 1 to 2 % slower than the best).  A product costs its launch, W's bytes at 11 TB/s, and its turns, one after
  // another, each as long as its own latency or as what the workgroups of a compute unit need together (lines: the blocks that the waves
  // take, and some); slices a second launch and the way of the sums out and back.  us, best and next:
  // 16 rows by 28,672 of 4,096 64 x 16 24, 128 x 32 in two 27; 64 by 6,144 of 2,048 64 x 32 9.7, 128 x 64 in eight 16; by 4,096 of 14,336 128 x 64
  // in eight 24, 64 x 32 in four 25; 256 by 28,672 of 4,096 256 x 64 81, 128 x 64 94; 32-bit rows, 32 by 2,048 of 2,048 64 x 32 in eight 8.1, 128 x 32 8.8
  const int t = dtype == kF32;
  float least = 0.f;
  Plan best{-1, 0, 0, 0, 0};
  for (int form = 0; form < (int)(sizeof kForms / sizeof *kForms); ++form) {
    const Form& f = kForms[form];
    if (f.busy[t] == 0.f || (silu && f.rows_w < 128 && (form >= kLinesForms || f.rows_w == 8))) continue;   // (silu: pairs of tiles a wave)
    for (int slices : {1, 2, 3, 4, 6, 8, 12, 16}) {
      const Plan p = laid_out(form, slices);
      const float groups = (float)p.n_tiles * p.m_tiles;
      if (p.slices != slices || slices > most_slices || (slices > 1 && groups * (slices - 1) > 512)) continue;
      const float each = groups * slices / 256, shared = each > 8 ? each + 0.5f : std::ceil(each);   // workgroups a compute unit
      const bool lines = form < kLinesForms;
      float us = (lines ? 3.1f : 2.1f) + (float)N * K * 4.8e-8f;
      if (lines) us += (std::min((float)p.turns, K / 32.f / f.step / slices) + 0.2f) * f.busy[t] * shared;
      else us += p.turns * std::max(f.alone[t], f.busy[t] * shared);
      if (slices > 1) us += 2.7f + slices * (float)M * N / 440e3f;
      if (best.form < 0 || us < least) least = us, best = p;
    }
  }
  return best;
}

template <typename T, int MT, int NT, int W, int U> static void lines(const Plan& p, const GemmArgs& a, hipStream_t stream) {
  static_assert(MT * NT * W <= 64, "the waves' sums fill LDS");
  const dim3 grid((unsigned)((p.n_tiles + 7) / 8 * 8 * p.m_tiles), (unsigned)p.slices);
  if constexpr (MT == 1 && std::is_same_v<T, bf16>) {
    if (a.parts || a.h) {
      hipLaunchKernelGGL((fp4_lines_kernel<T, MT, NT, W, U, true>), grid, dim3(W * kWave), 0, stream, a);
      return;
    }
  }
  hipLaunchKernelGGL((fp4_lines_kernel<T, MT, NT, W, U, false>), grid, dim3(W * kWave), 0, stream, a);
}
template <typename T, int MT, int NT, int B> static void tiles(const Plan& p, const GemmArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((fp4_tiles_kernel<T, MT, NT, B>), dim3((unsigned)((p.n_tiles + 7) / 8 * 8 * p.m_tiles), (unsigned)p.slices), dim3(256), 0, stream, a);
}

template <typename T> static void launch_by(const Plan& p, const GemmArgs& all, hipStream_t stream) {
  GemmArgs a = all;
  if (p.slices > 1) a.h = nullptr;   // (the pass behind the product does the norm)
  switch (p.form) {
    case 0: lines<T, 1, 4, 8, 1>(p, a, stream); break;
    case 1: lines<T, 1, 2, 8, 1>(p, a, stream); break;
    case 2: lines<T, 1, 1, 8, 2>(p, a, stream); break;
    case 3: lines<T, 2, 8, 4, 1>(p, a, stream); break;
    case 4: lines<T, 2, 4, 8, 1>(p, a, stream); break;
    case 5: lines<T, 1, 4, 4, 1>(p, a, stream); break;
    case 6: lines<T, 1, 8, 4, 1>(p, a, stream); break;
    default:
      if constexpr (std::is_same_v<T, float>) {
        if (p.form == 11) tiles<T, 2, 1, 4>(p, a, stream);
        else tiles<T, 2, 2, 4>(p, a, stream);
      } else {
        if (p.form == 7) tiles<T, 2, 1, 8>(p, a, stream);
        else if (p.form == 8) tiles<T, 2, 2, 8>(p, a, stream);
        else if (p.form == 9) tiles<T, 4, 2, 8>(p, a, stream);
        else tiles<T, 4, 4, 4>(p, a, stream);
      }
  }
  if (p.slices > 1 && all.h) {
    const int threads = std::min(1024, (a.N / 4 + kWave - 1) / kWave * kWave);
    hipLaunchKernelGGL(fp4_gemm_join_norm_kernel, dim3((unsigned)a.M), dim3(threads), 0, stream, all, p.slices);
  } else if (p.slices > 1) {
    const long long cells = (long long)a.M * (a.epilogue == 2 ? a.N / 2 : a.N);
    hipLaunchKernelGGL(fp4_gemm_join_kernel, dim3((unsigned)((cells + 255) / 256)), dim3(256), 0, stream, a, p.slices);
  }
}

}  // namespace gb

using namespace gb;

// floats of workspace with which k is divided; 0: it is not
extern "C" long long gb_fp4_gemm_floats(int M, int N, int K, int epilogue, int dtype) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan p = plan(M, N, K, epilogue == 2, dtype, 16);
  return p.slices > 1 ? (long long)p.slices * M * N : 0;
}

// tiles whose sums of squares a product that adds up to 8 rows leaves for the norm behind it; 0: it does not
extern "C" int gb_fp4_gemm_emit_parts(int M, int N) {
  return M > 0 && M <= kNormRows && N > 0 && N % 8 == 0 ? plan(M, N, 32, false, kBF16, 1).n_tiles : 0;
}

// What a product that adds a.w to the residual can do for the norm behind it: 0 nothing; 1 partial sums (the tiles above); 2, where it divides k and
// has its workspace, the whole norm (h given without sums).
extern "C" int gb_fp4_gemm_emit_mode(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if (M <= kNormRows) return N % 8 == 0 ? 1 : 0;
  return N % 4 == 0 && N <= kNormColumns && plan(M, N, K, false, kBF16, 16).slices > 1 ? 2 : 0;
}

// with what a product does for norms (GemmArgs)
extern "C" int gb_fp4_gemm_norms(const void* x, int dtype, int ldx, const void* codes, const void* scales, int scale_stride, void* out, int out_dtype,
                                 int ldo, int M, int N, int K, int epilogue, float* workspace, long long workspace_floats, const void* gamma,
                                 int gamma_dtype, void* h, int ldh, float* sums, const float* parts, int n_parts, float eps, hipStream_t stream) {
  GB_REQUIRE(M >= 0 && N > 0 && K > 0 && K % 32 == 0, "fp4_gemm: bad sizes M=%d N=%d K=%d", M, N, K);
  GB_REQUIRE(epilogue >= 0 && epilogue <= 2 && (epilogue != 2 || N % 2 == 0), "fp4_gemm: epilogue %d of %d columns", epilogue, N);
  GB_REQUIRE(epilogue != 1 || out_dtype == kF32, "fp4_gemm: accumulation is into a 32-bit result");
  GB_REQUIRE(ldx >= K && ldo >= (epilogue == 2 ? N / 2 : N), "fp4_gemm: row strides %d, %d are shorter than the rows", ldx, ldo);
  GB_REQUIRE(scale_stride >= K / 32 && scale_stride % 16 == 0 && ((uintptr_t)codes & 15) == 0 && ((uintptr_t)scales & 15) == 0,
             "fp4_gemm: codes and scales begin at 16-byte words, rows of scales are multiples of 16");
  GB_REQUIRE((dtype == kF32 || dtype == kBF16) && (out_dtype == kF32 || out_dtype == kBF16), "fp4_gemm: unknown dtype %d or %d", dtype, out_dtype);
  GB_REQUIRE(!h || (dtype == kBF16 && epilogue == 1 && M <= (sums ? kNormRows : INT32_MAX) && N % (sums ? 8 : 4) == 0 && (uintptr_t)out % 16 == 0 && ldo % 4 == 0 &&
                    (uintptr_t)h % 8 == 0 && ldh % 4 == 0 && ldh >= N && gamma && (gamma_dtype == kF32 || gamma_dtype == kBF16)),
             "fp4_gemm: a norm is prepared by products that add bfloat16 rows (up to %d, or with k divided), of a multiple of 8 (4) columns in whole words",
             kNormRows);
  GB_REQUIRE(!parts || (dtype == kBF16 && epilogue != 1 && M <= kNormRows && n_parts > 0 && n_parts < (1 << 24) && (uintptr_t)parts % 16 == 0), "fp4_gemm: a norm's sums go with up to %d bfloat16 rows", kNormRows);
  if (M == 0) return 0;
  Plan p = plan(M, N, K, epilogue == 2, dtype, 16);
  if (p.slices > 1 && (!workspace || workspace_floats < (long long)p.slices * M * N)) p = plan(M, N, K, epilogue == 2, dtype, 1);   // slower, not refused
  GB_REQUIRE(!h || sums || (p.slices > 1 && N <= kNormColumns), "fp4_gemm: a norm of rows whose product does not divide k, or of more than %d columns", kNormColumns);
  GB_REQUIRE((long long)(p.n_tiles + 7) * p.m_tiles < (1ll << 31) && (long long)M * N < (1ll << 38), "fp4_gemm: %d x %d is too much for one launch", M, N);
  const int e = out_dtype == kF32 ? 16 : 8;   // bytes of four columns
  const GemmArgs a{x, (const uint8_t*)codes, (const uint8_t*)scales, out, p.slices > 1 ? workspace : nullptr, parts, gamma,
                   (bf16*)h, sums, n_parts, gamma_dtype == kF32, ldh, eps, ldx, ldo, M, N, K / 32, scale_stride,
                   p.n_tiles, p.m_tiles, p.turns, epilogue, out_dtype == kF32, (uintptr_t)out % e == 0 && ldo % 4 == 0};
  if (dtype == kF32) launch_by<float>(p, a, stream);
  else launch_by<bf16>(p, a, stream);
  return launched("fp4_gemm");
}

extern "C" int gb_fp4_gemm(const void* x, int dtype, int ldx, const void* codes, const void* scales, int scale_stride, void* out, int out_dtype,
                           int ldo, int M, int N, int K, int epilogue, float* workspace, long long workspace_floats, hipStream_t stream) {
  return gb_fp4_gemm_norms(x, dtype, ldx, codes, scales, scale_stride, out, out_dtype, ldo, M, N, K, epilogue, workspace, workspace_floats, nullptr, kF32,
                           nullptr, 0, nullptr, nullptr, 0, 0.f, stream);
}

GB_TAPED(gb_fp4_gemm)
GB_TAPED(gb_fp4_gemm_norms)
GB_DEFINE_LAST_ERROR
