// Four-bit pages (fp4.h): keys and values stored into them, with the rotation of queries and keys on the way, and read back;
// and matrices quantized to the same blocks.
//
// All of it is bound by memory, or, for the rows of a decode step, by the launch: a few operations a byte.
#include "fp4.h"

namespace gb {

// Largest of the four lanes that hold a block's quarters, 16 lanes apart; the lanes of a quarter hold 16 tokens.
__device__ __forceinline__ uint32_t quarters_max(uint32_t v) {
  const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return max(b[0], b[1]);
}
__device__ __forceinline__ uint32_t largest8(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  return m;
}

struct StoreArgs {
  const void* qkv;
  void* q;
  const float *cosv, *sinv;
  const int32_t* slots;
  uint8_t *k, *v;
  int stride, q_stride, n, nh, nkv, hd, page, pages, wide, q_wide, cs_wide;
  int kv_blocks;   // workgroups that store; the others turn queries
};

// Keys and values: a wave takes one block of 32 channels of 16 tokens, lane l tokens l % 16 and the channels' quarter l / 16, so that
// what 16 neighbouring tokens bring lies side by side in both kinds of pages: a store of keys fills 256 bytes, one of values four
// runs of 16.  (A lane a whole block would have the rows' reads in whole lines, and the values' bytes in stores of one token each.)
// Queries: a lane takes 8 pairs (i, i + hd / 2) and may write where it read.
template <typename T>
__global__ __launch_bounds__(256) void fp4_store_kernel(StoreArgs a) {
  const int lane = threadIdx.x % kWave, half = a.hd / 2;
  if ((int)blockIdx.x < a.kv_blocks) {
    const int nb = a.hd / kFp4Block, units = 2 * a.nkv * nb;
    const int wave = blockIdx.x * 4 + threadIdx.x / kWave;
    const int unit = wave % units, group = wave / units;
    const int t = group * 16 + lane % 16, quarter = lane / 16;
    if (group * 16 >= a.n) return;
    const int slot = t < a.n ? a.slots[t] : -1;
    const bool stored = slot >= 0 && slot / a.page < a.pages;
    const int row = t < a.n ? t : a.n - 1;
    const int head = unit / nb, b = unit % nb;   // keys' heads, then values'
    const T* src = (const T*)a.qkv + (size_t)row * a.stride + (size_t)(a.nh + head) * a.hd;
    const int c = b * kFp4Block + quarter * 8;
    float x[8];
    load8(src + c, a.wide, x);
    if (head < a.nkv && a.cosv) {
      const bool low = c < half;
      float other[8], cs[8], sn[8];
      load8(src + (low ? c + half : c - half), a.wide, other);
      const size_t at = (size_t)row * half + (low ? c : c - half);
      load8(a.cosv + at, a.cs_wide, cs);
      load8(a.sinv + at, a.cs_wide, sn);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = low ? turned_lo(x[i], other[i], cs[i], sn[i]) : turned_hi(other[i], x[i], cs[i], sn[i]);
    }
    const uint32_t byte = fp4_scale_byte(quarters_max(largest8(x)));
    uint32_t word = fp4_pack8(x, fp4_unit(byte));
    const int page = slot / a.page, off = slot % a.page;
    const size_t block = fp4_block_bytes(a.page);
    if (head < a.nkv) {
      if (!stored) return;
      uint8_t* dst = a.k + (((size_t)page * a.nkv + head) * nb + b) * block;
      *reinterpret_cast<uint32_t*>(dst + off * 16 + quarter * 4) = word;
      if (quarter == 0) dst[16 * a.page + fp4_key_scale_place(off)] = (uint8_t)byte;
    } else {
      // bytes of channels (i, i + 16): quarters 0 and 2 have the halves of rows 0..7, quarters 1 and 3 of rows 8..15; after the
      // exchange every lane has four rows to write
      const uint32_t theirs = __shfl_xor(word, 32, kWave);
      const uint32_t lo = quarter < 2 ? word : theirs, hi = quarter < 2 ? theirs : word;
      const int first = (quarter & 1) * 8 + (quarter >> 1) * 4, shift = (quarter >> 1) * 16;
      if (!stored) return;
      uint8_t* dst = a.v + (((size_t)page * a.nkv + head - a.nkv) * nb + b) * block + off;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        dst[(size_t)(first + i) * a.page] = (uint8_t)(((lo >> (shift + 4 * i)) & 15u) | (((hi >> (shift + 4 * i)) & 15u) << 4));
      if (quarter == 0) dst[(size_t)16 * a.page] = (uint8_t)byte;
    }
    return;
  }
  const int pieces = half / 8;
  const long long item = (long long)(blockIdx.x - a.kv_blocks) * 256 + threadIdx.x;
  const int t = (int)(item / (a.nh * pieces)), rest = (int)(item % (a.nh * pieces));
  if (t >= a.n) return;
  const int head = rest / pieces, c = rest % pieces * 8;
  const T* src = (const T*)a.qkv + (size_t)t * a.stride + (size_t)head * a.hd + c;
  T* dst = (T*)a.q + (size_t)t * a.q_stride + (size_t)head * a.hd + c;
  float x0[8], x1[8];
  load8(src, a.wide, x0);
  load8(src + half, a.wide, x1);
  if (a.cosv) {
    float cs[8], sn[8], y0[8], y1[8];
    load8(a.cosv + (size_t)t * half + c, a.cs_wide, cs);
    load8(a.sinv + (size_t)t * half + c, a.cs_wide, sn);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y0[i] = turned_lo(x0[i], x1[i], cs[i], sn[i]);
      y1[i] = turned_hi(x0[i], x1[i], cs[i], sn[i]);
    }
    store8(dst, a.q_wide, y0);
    store8(dst + half, a.q_wide, y1);
  } else {
    store8(dst, a.q_wide, x0);
    store8(dst + half, a.q_wide, x1);
  }
}

// Rows back from their slots: the lanes of a wave as above.  A lane takes eight channels, a word of a key, or a byte of eight rows of
// values of which it needs one half.
template <typename T>
__global__ __launch_bounds__(256) void fp4_load_kernel(const int32_t* __restrict__ slots, const uint8_t* __restrict__ k_pages,
                                                      const uint8_t* __restrict__ v_pages, T* __restrict__ k, T* __restrict__ v,
                                                      int k_stride, int v_stride, int n, int nkv, int hd, int page, int pages,
                                                      int k_wide, int v_wide) {
  const int nb = hd / kFp4Block, units = 2 * nkv * nb, lane = threadIdx.x % kWave;
  const int wave = blockIdx.x * 4 + threadIdx.x / kWave;
  const int unit = wave % units, t = wave / units * 16 + lane % 16, quarter = lane / 16;
  if (t >= n) return;
  const int slot = slots[t];
  if (slot < 0 || slot / page >= pages) return;
  const int head = unit / nb % nkv, b = unit % nb, off = slot % page;
  const uint8_t* block = (unit < nkv * nb ? k_pages : v_pages) + (((size_t)(slot / page) * nkv + head) * nb + b) * fp4_block_bytes(page);
  uint32_t word = 0;
  float unit_of;
  if (unit < nkv * nb) {
    word = *reinterpret_cast<const uint32_t*>(block + off * 16 + quarter * 4);
    unit_of = fp4_unit(block[16 * page + fp4_key_scale_place(off)]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) word |= ((uint32_t)block[((quarter & 1) * 8 + i) * page + off] >> (quarter >= 2 ? 4 : 0) & 15u) << (4 * i);
    unit_of = fp4_unit(block[16 * page + off]);
  }
  const bf16x8 y = fp4_unpack8(word, unit_of);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)y[i];
  const size_t col = (size_t)head * hd + b * kFp4Block + quarter * 8;
  if (unit < nkv * nb) store8(k + (size_t)t * k_stride + col, k_wide, x);
  else store8(v + (size_t)t * v_stride + col, v_wide, x);
}

// Matrices: four lanes a block, neighbours, so that rows are read and codes written in whole lines.
template <typename T>
__global__ __launch_bounds__(256) void fp4_quantize_kernel(const T* __restrict__ w, int stride, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales, int n, int blocks, int scale_stride, int wide) {
  const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
  const int quarter = (int)(item & 3), b = (int)((item >> 2) % scale_stride);
  const long long row = (item >> 2) / scale_stride;
  if (row >= n) return;   // (the lanes of a block leave together)
  if (b >= blocks) {
    if (quarter == 0) scales[row * scale_stride + b] = 0;
    return;
  }
  float x[8];
  load8(w + row * stride + b * kFp4Block + quarter * 8, wide, x);
  uint32_t m = largest8(x);
  m = max(m, (uint32_t)__shfl_xor(m, 1, 4));
  m = max(m, (uint32_t)__shfl_xor(m, 2, 4));
  const uint32_t byte = fp4_scale_byte(m);
  *reinterpret_cast<uint32_t*>(codes + row * (blocks * 16) + b * 16 + quarter * 4) = fp4_pack8(x, fp4_unit(byte));
  if (quarter == 0) scales[row * scale_stride + b] = (uint8_t)byte;
}

// Matrices back to bf16 (or 32-bit) rows: a lane a word.
template <typename T>
__global__ __launch_bounds__(256) void fp4_expand_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                        T* __restrict__ w, int n, int blocks, int scale_stride) {
  const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = item / (blocks * 4);
  const int word = (int)(item % (blocks * 4));
  if (row >= n) return;
  const bf16x8 y = fp4_unpack8(*reinterpret_cast<const uint32_t*>(codes + row * (blocks * 16) + word * 4),
                               fp4_unit(scales[row * scale_stride + word / 4]));
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)y[i];
  store8(w + (row * blocks * 4 + word) * 8, true, x);
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace gb

using namespace gb;

extern "C" int gb_fp4_store(const void* qkv, int dtype, int stride, void* q, int q_stride, const float* cosv, const float* sinv,
                            const int32_t* slots, void* k_pages, void* v_pages, int n, int nh, int nkv, int hd, int page, int pages,
                            hipStream_t stream) {
  GB_REQUIRE(n >= 0 && nh >= 0 && nkv >= 0 && hd > 0 && hd % 32 == 0, "fp4_store: bad sizes n=%d nh=%d nkv=%d hd=%d", n, nh, nkv, hd);
  GB_REQUIRE((long long)(nh + 2ll * nkv) * hd <= stride, "fp4_store: row stride %d is shorter than the stacked heads", stride);
  GB_REQUIRE(!slots || (k_pages && v_pages && page > 0 && page % 16 == 0 && pages > 0), "fp4_store: slots without pages of a multiple of 16 slots");
  GB_REQUIRE(!cosv == !sinv, "fp4_store: cosines and sines go together");
  GB_REQUIRE(dtype == kF32 || dtype == kBF16, "fp4_store: unknown dtype %d", dtype);
  const int e = dtype == kF32 ? 4 : 2;
  const bool turns = q && nh > 0 && (cosv || q != qkv);
  const long long waves = slots ? (long long)((n + 15) / 16) * 2 * nkv * (hd / 32) : 0;
  const long long kv = (waves + 3) / 4, items = turns ? (long long)n * nh * (hd / 16) : 0, blocks = kv + (items + 255) / 256;
  if (n == 0 || blocks == 0) return 0;
  GB_REQUIRE(blocks < (1ll << 31) && waves < (1ll << 31), "fp4_store: %d rows are too many for one launch", n);
  StoreArgs a{qkv, q, cosv, sinv, slots, (uint8_t*)k_pages, (uint8_t*)v_pages, stride, q_stride, n, nh, nkv, hd, page, pages,
              aligned16(qkv) && (size_t)stride * e % 16 == 0, aligned16(q) && (size_t)q_stride * e % 16 == 0,
              aligned16(cosv) && aligned16(sinv), (int)kv};
  if (dtype == kF32) hipLaunchKernelGGL(fp4_store_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(fp4_store_kernel<bf16>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return launched("fp4_store");
}

extern "C" int gb_fp4_load(const int32_t* slots, const void* k_pages, const void* v_pages, void* k, int k_stride, void* v, int v_stride,
                           int dtype, int n, int nkv, int hd, int page, int pages, hipStream_t stream) {
  GB_REQUIRE(n >= 0 && nkv > 0 && hd > 0 && hd % 32 == 0 && page > 0 && page % 16 == 0 && pages > 0, "fp4_load: bad sizes n=%d nkv=%d hd=%d page=%d", n,
             nkv, hd, page);
  GB_REQUIRE(nkv * (long long)hd <= k_stride && nkv * (long long)hd <= v_stride, "fp4_load: row strides %d, %d are shorter than the heads", k_stride,
             v_stride);
  GB_REQUIRE(dtype == kF32 || dtype == kBF16, "fp4_load: unknown dtype %d", dtype);
  if (n == 0) return 0;
  const long long waves = (long long)((n + 15) / 16) * 2 * nkv * (hd / 32), blocks = (waves + 3) / 4;
  GB_REQUIRE(waves < (1ll << 31), "fp4_load: %d rows are too many for one launch", n);
  const int e = dtype == kF32 ? 4 : 2;
  const int kw = aligned16(k) && (size_t)k_stride * e % 16 == 0, vw = aligned16(v) && (size_t)v_stride * e % 16 == 0;
  if (dtype == kF32)
    hipLaunchKernelGGL(fp4_load_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, stream, slots, (const uint8_t*)k_pages,
                       (const uint8_t*)v_pages, (float*)k, (float*)v, k_stride, v_stride, n, nkv, hd, page, pages, kw, vw);
  else
    hipLaunchKernelGGL(fp4_load_kernel<bf16>, dim3((unsigned)blocks), dim3(256), 0, stream, slots, (const uint8_t*)k_pages,
                       (const uint8_t*)v_pages, (bf16*)k, (bf16*)v, k_stride, v_stride, n, nkv, hd, page, pages, kw, vw);
  return launched("fp4_load");
}

extern "C" int gb_fp4_quantize(const void* w, int dtype, int stride, void* codes, void* scales, int n, int k, int scale_stride,
                               hipStream_t stream) {
  GB_REQUIRE(n >= 0 && k > 0 && k % 32 == 0 && stride >= k && scale_stride >= k / 32, "fp4_quantize: bad sizes n=%d k=%d", n, k);
  GB_REQUIRE(dtype == kF32 || dtype == kBF16, "fp4_quantize: unknown dtype %d", dtype);
  if (n == 0) return 0;
  const long long blocks = ((long long)n * scale_stride * 4 + 255) / 256;
  GB_REQUIRE(blocks < (1ll << 31), "fp4_quantize: %d rows of %d are too many for one launch", n, k);
  const int wide = aligned16(w) && (size_t)stride * (dtype == kF32 ? 4 : 2) % 16 == 0;
  if (dtype == kF32)
    hipLaunchKernelGGL(fp4_quantize_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, stream, (const float*)w, stride, (uint8_t*)codes,
                       (uint8_t*)scales, n, k / 32, scale_stride, wide);
  else
    hipLaunchKernelGGL(fp4_quantize_kernel<bf16>, dim3((unsigned)blocks), dim3(256), 0, stream, (const bf16*)w, stride, (uint8_t*)codes,
                       (uint8_t*)scales, n, k / 32, scale_stride, wide);
  return launched("fp4_quantize");
}

extern "C" int gb_fp4_expand(const void* codes, const void* scales, void* w, int dtype, int n, int k, int scale_stride, hipStream_t stream) {
  GB_REQUIRE(n >= 0 && k > 0 && k % 32 == 0 && scale_stride >= k / 32 && aligned16(w), "fp4_expand: bad sizes n=%d k=%d, or rows that do not begin at 16 bytes", n, k);
  GB_REQUIRE(dtype == kF32 || dtype == kBF16, "fp4_expand: unknown dtype %d", dtype);
  if (n == 0) return 0;
  const long long blocks = ((long long)n * (k / 8) + 255) / 256;
  GB_REQUIRE(blocks < (1ll << 31), "fp4_expand: %d rows of %d are too many for one launch", n, k);
  if (dtype == kF32)
    hipLaunchKernelGGL(fp4_expand_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, stream, (const uint8_t*)codes, (const uint8_t*)scales,
                       (float*)w, n, k / 32, scale_stride);
  else
    hipLaunchKernelGGL(fp4_expand_kernel<bf16>, dim3((unsigned)blocks), dim3(256), 0, stream, (const uint8_t*)codes, (const uint8_t*)scales,
                       (bf16*)w, n, k / 32, scale_stride);
  return launched("fp4_expand");
}

GB_TAPED(gb_fp4_store)
GB_TAPED(gb_fp4_load)
GB_TAPED(gb_fp4_quantize)
GB_TAPED(gb_fp4_expand)
GB_DEFINE_LAST_ERROR
