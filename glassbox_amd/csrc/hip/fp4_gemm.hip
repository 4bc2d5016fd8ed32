// Products with four-bit weights (fp4.h): out (+)= a . W^T, or silu(a . gate^T) * (a . up^T) of a stack of both.
//
// Few rows: what bounds it is W's bytes, 17 / 32 of one a number.  W is the left operand of 16 x 16 x 32 products, so that a lane's
// numbers are 32 neighbours of one row of W with one scale: 16 bytes and a byte.  They become bf16 in registers, two an instruction,
// exactly, and never see LDS.  Waves of a workgroup take every W-th 128 numbers of k and are added up through LDS in their order.
// The rows of a come from memory to every wave (they are in L2): NT tiles of 16 rows of W share what a wave reads of them.
// 32-bit rows count as three bf16 terms (fp4.h): the products stay exact, their sums are in 32 bits either way.
#include "fp4.h"

#include <algorithm>

namespace gb {

struct GemmArgs {
  const void* x;
  const uint8_t *codes, *scales;
  void* out;
  int ldx, ldo, M, N, blocks, scale_stride, n_tiles, m_tiles, epilogue, out32, x_wide;   // epilogue 0 store, 1 add, 2 silu(gate) * up
};

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ void put(const GemmArgs& a, int m, int n, int limit, const f32x4& v) {
  const size_t at = (size_t)m * a.ldo + n;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < limit) {
      if (a.out32) {
        float* o = (float*)a.out + at + i;
        *o = a.epilogue == 1 ? *o + v[i] : v[i];
      } else {
        ((bf16*)a.out)[at + i] = (bf16)v[i];
      }
    }
}

// T the rows' type, MT tiles of 16 rows of a, NT of 16 rows of W (with silu every other one of the up half), W waves
template <typename T, int MT, int NT, int W>
__global__ __launch_bounds__(W * kWave) void fp4_gemm_kernel(GemmArgs a) {
  constexpr int SP = kFp4Terms<T>;
  const int lane = threadIdx.x % kWave, r = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // the row tiles of one tile of W follow each other on one XCD (workgroups go to the eight in turn), whose L2 then has it
  const int turn = blockIdx.x / 8, nt = turn / a.m_tiles * 8 + blockIdx.x % 8, mt0 = turn % a.m_tiles * 16 * MT;
  if (nt >= a.n_tiles) return;
  const bool silu = a.epilogue == 2;
  const int half = a.N / 2;
  int row0[NT], limit[NT];
  const uint8_t *codes[NT], *scales[NT];
#pragma unroll
  for (int p = 0; p < NT; ++p) {
    row0[p] = silu ? (p & 1 ? half : 0) + (nt * (NT / 2) + p / 2) * 16 : (nt * NT + p) * 16;
    limit[p] = silu && !(p & 1) ? half : a.N;
    const int row = min(row0[p] + r, limit[p] - 1);
    codes[p] = a.codes + (size_t)row * a.blocks * 16 + g * 16;
    scales[p] = a.scales + (size_t)row * a.scale_stride;
  }
  const T* x[MT];
  bool has[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int m = mt0 + 16 * t + r;
    has[t] = m < a.M;
    x[t] = (const T*)a.x + (size_t)min(m, a.M - 1) * a.ldx + g * kFp4Block;
  }
  f32x4 acc[NT][MT];
#pragma unroll
  for (int p = 0; p < NT; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[p][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int chunks = (a.blocks + 3) / 4;
  u32x4 next[NT];
  uint32_t nexts[NT];
  auto fetch = [&](int c) {
    const bool in = 4 * c + g < a.blocks;
#pragma unroll
    for (int p = 0; p < NT; ++p) {
      next[p] = in ? *reinterpret_cast<const u32x4*>(codes[p] + (size_t)c * 64) : u32x4{0, 0, 0, 0};
      nexts[p] = *reinterpret_cast<const uint32_t*>(scales[p] + 4 * c);
    }
  };
  if (wave < chunks) fetch(wave);
  for (int c = wave; c < chunks; c += W) {
    u32x4 now[NT];
    float unit[NT];
#pragma unroll
    for (int p = 0; p < NT; ++p) now[p] = next[p], unit[p] = fp4_unit(nexts[p] >> (8 * g) & 255u);
    const bool in = 4 * c + g < a.blocks;
    bf16x8 xf[MT][4][SP];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float v[8] = {};
        if (in && has[t]) load8(x[t] + (size_t)c * 128 + 8 * w, a.x_wide, v);
        fp4_terms<SP>(v, xf[t][w]);
      }
    if (c + W < chunks) fetch(c + W);
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int p = 0; p < NT; ++p) {
        const bf16x8 kf = fp4_unpack8(now[p][w], unit[p]);
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int q = 0; q < SP; ++q) acc[p][t] = mfma(kf, xf[t][w][q], acc[p][t]);
      }
  }

  __shared__ f32x4 part[W][NT * MT][kWave];
#pragma unroll
  for (int p = 0; p < NT; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t) part[wave][p * MT + t][lane] = acc[p][t];
  __syncthreads();
  auto total = [&](int tile) {
    f32x4 v = part[0][tile][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += part[w][tile][lane];
    return v;
  };
  if (silu) {
    for (int u = wave; u < NT / 2 * MT; u += W) {
      const int p = u / MT * 2, t = u % MT, m = mt0 + 16 * t + r;
      const f32x4 gate = total(p * MT + t), up = total((p + 1) * MT + t);
      f32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = silu_times(gate[i], up[i]);
      if (m < a.M) put(a, m, (nt * (NT / 2) + p / 2) * 16 + 4 * g, half, v);
    }
  } else {
    for (int u = wave; u < NT * MT; u += W) {
      const int p = u / MT, t = u % MT, m = mt0 + 16 * t + r;
      const f32x4 v = total(u);
      if (m < a.M) put(a, m, (nt * NT + p) * 16 + 4 * g, a.N, v);
    }
  }
}

template <typename T, int MT, int NT, int W> static void launch(GemmArgs a, hipStream_t stream) {
  const int rows = a.epilogue == 2 ? a.N / 2 : a.N, per = 16 * (a.epilogue == 2 ? NT / 2 : NT);
  a.n_tiles = (rows + per - 1) / per;
  a.m_tiles = (a.M + 16 * MT - 1) / (16 * MT);
  hipLaunchKernelGGL((fp4_gemm_kernel<T, MT, NT, W>), dim3((unsigned)((a.n_tiles + 7) / 8 * 8 * a.m_tiles)), dim3(W * kWave), 0, stream, a);
}

template <typename T> static void launch_by(const GemmArgs& a, hipStream_t stream) {
  const int tiles = (a.N + 15) / 16;
  const bool silu = a.epilogue == 2;
  if (a.M <= 16) {
    if (tiles >= 2048) launch<T, 1, 4, 4>(a, stream);
    else if (silu || tiles >= 512) launch<T, 1, 2, 8>(a, stream);
    else launch<T, 1, 1, 8>(a, stream);
  } else if (a.M <= 32) {
    if (tiles >= 1024) launch<T, 2, 4, 4>(a, stream);
    else launch<T, 2, 2, 4>(a, stream);
  } else {
    if (tiles >= 1024 || a.M > 128) launch<T, 4, 4, 4>(a, stream);
    else launch<T, 4, 2, 4>(a, stream);
  }
}

}  // namespace gb

using namespace gb;

extern "C" int gb_fp4_gemm(const void* x, int dtype, int ldx, const void* codes, const void* scales, int scale_stride, void* out, int out_dtype,
                           int ldo, int M, int N, int K, int epilogue, hipStream_t stream) {
  GB_REQUIRE(M >= 0 && N > 0 && K > 0 && K % 32 == 0, "fp4_gemm: bad sizes M=%d N=%d K=%d", M, N, K);
  GB_REQUIRE(epilogue >= 0 && epilogue <= 2 && (epilogue != 2 || N % 2 == 0), "fp4_gemm: epilogue %d of %d columns", epilogue, N);
  GB_REQUIRE(epilogue != 1 || out_dtype == kF32, "fp4_gemm: accumulation is into a 32-bit result");
  GB_REQUIRE(ldx >= K && ldo >= (epilogue == 2 ? N / 2 : N), "fp4_gemm: row strides %d, %d are shorter than the rows", ldx, ldo);
  GB_REQUIRE(scale_stride >= K / 32 && scale_stride % 16 == 0 && ((uintptr_t)codes & 15) == 0 && ((uintptr_t)scales & 15) == 0,
             "fp4_gemm: codes and scales begin at 16-byte words, rows of scales are multiples of 16");
  GB_REQUIRE((dtype == kF32 || dtype == kBF16) && (out_dtype == kF32 || out_dtype == kBF16), "fp4_gemm: unknown dtype %d or %d", dtype, out_dtype);
  if (M == 0) return 0;
  GB_REQUIRE((long long)((N + 15) / 16 + 8) * ((M + 15) / 16) < (1ll << 31), "fp4_gemm: %d x %d is too much for one launch", M, N);
  const int e = dtype == kF32 ? 4 : 2;
  GemmArgs a{x, (const uint8_t*)codes, (const uint8_t*)scales, out, ldx, ldo, M, N, K / 32, scale_stride, 0, 0, epilogue, out_dtype == kF32,
             ((uintptr_t)x & 15) == 0 && (size_t)ldx * e % 16 == 0};
  if (dtype == kF32) launch_by<float>(a, stream);
  else launch_by<bf16>(a, stream);
  return launched("fp4_gemm");
}

GB_TAPED(gb_fp4_gemm)
GB_DEFINE_LAST_ERROR
