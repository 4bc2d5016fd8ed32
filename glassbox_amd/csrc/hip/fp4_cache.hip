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

// Four neighbouring lanes hold four bytes each: lane i gets the four bytes i, in the order of the lanes.
__device__ __forceinline__ uint32_t turn_bytes(uint32_t w, int lane) {
  const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp((int)w, 0xb1, 0xf, 0xf, true);   // of lane ^ 1
  w = lane & 1 ? __builtin_amdgcn_perm(w, a, 0x07030501u) : __builtin_amdgcn_perm(a, w, 0x06020400u);
  const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp((int)w, 0x4e, 0xf, 0xf, true);   // of lane ^ 2
  return lane & 2 ? __builtin_amdgcn_perm(w, b, 0x07060302u) : __builtin_amdgcn_perm(b, w, 0x05040100u);
}
// Whether the slots of this lane and its three neighbours (tokens 4 i .. 4 i + 3) are four in a row from a multiple of four on: their
// bytes in a row of values are then one word.  All lanes take part.
__device__ __forceinline__ bool quad_in_a_row(int slot, bool stored, int lane) {
  const int first = __builtin_amdgcn_mov_dpp(slot, 0x00, 0xf, 0xf, true);
  const bool fits = stored && slot - (lane & 3) == first && (first & 3) == 0;
  return (__ballot(fits) >> (lane & ~3) & 15) == 15;
}

struct StoreArgs {
  const void* qkv;
  void* q;
  const float *cosv, *sinv;
  const int32_t* slots;
  uint8_t *k, *v;
  int stride, q_stride, n, nh, nkv, hd, page, pages, wide, q_wide, cs_wide;
  int kv_blocks, k_units, v_units;   // workgroups that store, the others turn queries; units of 16 tokens' keys and of their values
};

// Keys and values: a wave takes 16 tokens, lane l token l % 16 and of a block of 32 channels the quarter l / 16, so that what neighbouring
// tokens bring lies side by side in both kinds of pages: a store of keys fills 256 bytes, and so does one of values where the tokens' slots
// follow each other (their bytes are exchanged between four lanes).  Keys of heads of 64 channels and multiples go two blocks at a time,
// (i, i + hd / 2).  A lane takes kHeads heads, which share their angles, one after the other: 6,151 rows of 8 kv heads of 128 in 11 us, a head at a
// time and values byte by byte in 21; with the queries of 32 heads 27 and 39.  The few rows of a decode step take one: 3.6 us, four 4.6.
// Queries: a lane takes 8 pairs (i, i + hd / 2) and may write where it read.
template <typename T, bool PAIRS, int kHeads>
__global__ __launch_bounds__(256) void fp4_store_kernel(StoreArgs a) {
  const int lane = threadIdx.x % kWave, half = a.hd / 2;
  if ((int)blockIdx.x < a.kv_blocks) {
    const int nb = a.hd / kFp4Block, units = a.k_units + a.v_units;
    const int wave = blockIdx.x * 4 + threadIdx.x / kWave;
    int unit = wave % units;
    const int group = wave / units, t = group * 16 + lane % 16, quarter = lane / 16;
    if (group * 16 >= a.n) return;
    const int row = min(t, a.n - 1), slot = t < a.n ? a.slots[t] : -1;
    const bool stored = slot >= 0 && slot / a.page < a.pages;
    const int page = stored ? slot / a.page : 0, off = stored ? slot % a.page : 0;
    const size_t block = fp4_block_bytes(a.page), head_bytes = block * nb;
    if (unit < a.k_units) {
      constexpr int B = PAIRS ? 2 : 1;
      const int per = PAIRS ? nb / 2 : nb, head0 = unit / per * kHeads, b = unit % per;
      const int c = b * kFp4Block + quarter * 8;                       // and with PAIRS c + half
      const bool low = PAIRS || c < half;
      const int other = low ? c + half : c - half, angle = low ? c : other;
      const T* src = (const T*)a.qkv + (size_t)row * a.stride + (size_t)a.nh * a.hd;
      uint8_t* dst = a.k + (size_t)page * a.nkv * head_bytes + (size_t)b * block;
      float cs[8], sn[8], x[kHeads][8], y[kHeads][8];
      if (a.cosv) {
        load8(a.cosv + (size_t)row * half + angle, a.cs_wide, cs);
        load8(a.sinv + (size_t)row * half + angle, a.cs_wide, sn);
      }
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        const T* p = src + (size_t)min(head0 + h, a.nkv - 1) * a.hd;
        load8(p + c, a.wide, x[h]);
        if (PAIRS || a.cosv) load8(p + other, a.wide, y[h]);
      }
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        if (head0 + h >= a.nkv) return;
        if (a.cosv) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float lo = low ? x[h][i] : y[h][i], hi = low ? y[h][i] : x[h][i];
            const float first = turned_lo(lo, hi, cs[i], sn[i]), second = turned_hi(lo, hi, cs[i], sn[i]);
            x[h][i] = low ? first : second;
            y[h][i] = second;
          }
        }
#pragma unroll
        for (int k = 0; k < B; ++k) {
          const float(&z)[8] = k ? y[h] : x[h];
          const uint32_t byte = fp4_scale_byte(quarters_max(largest8(z))), word = fp4_pack8(z, fp4_unit(byte));
          uint8_t* to = dst + (size_t)(head0 + h) * head_bytes + (size_t)(k * (nb / 2)) * block;
          if (stored) {
            *reinterpret_cast<uint32_t*>(to + off * 16 + quarter * 4) = word;
            if (quarter == 0) to[16 * a.page + fp4_key_scale_place(off)] = (uint8_t)byte;
          }
        }
      }
      return;
    }
    unit -= a.k_units;
    const int head0 = unit / nb * kHeads, b = unit % nb;
    const T* src = (const T*)a.qkv + (size_t)row * a.stride + (size_t)(a.nh + a.nkv) * a.hd + b * kFp4Block + quarter * 8;
    uint8_t* dst = a.v + (size_t)page * a.nkv * head_bytes + (size_t)b * block;
    const bool words = quad_in_a_row(slot, stored, lane);
    float x[kHeads][8];
#pragma unroll
    for (int h = 0; h < kHeads; ++h) load8(src + (size_t)min(head0 + h, a.nkv - 1) * a.hd, a.wide, x[h]);
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      if (head0 + h >= a.nkv) return;
      const uint32_t byte = fp4_scale_byte(quarters_max(largest8(x[h]))), word = fp4_pack8(x[h], fp4_unit(byte));
      // bytes of channels (i, i + 16): quarters 0 and 2 have the halves of rows 0..7, quarters 1 and 3 of rows 8..15; after the exchange every
      // lane has four rows of its token
      const uint32_t theirs = __shfl_xor(word, 32, kWave);
      const int shift = (quarter >> 1) * 16, first = (quarter & 1) * 8 + (quarter >> 1) * 4;
      const uint32_t lo = (quarter < 2 ? word : theirs) >> shift, hi = (quarter < 2 ? theirs : word) >> shift;
      uint32_t four = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) four |= ((lo >> (4 * i) & 15u) | (hi >> (4 * i) & 15u) << 4) << (8 * i);
      const uint32_t turned = turn_bytes(four, lane);
      uint8_t* to = dst + (size_t)(head0 + h) * head_bytes;
      if (words) {
        *reinterpret_cast<uint32_t*>(to + (size_t)(first + (lane & 3)) * a.page + (off & ~3)) = turned;
      } else if (stored) {
#pragma unroll
        for (int i = 0; i < 4; ++i) to[(size_t)(first + i) * a.page + off] = (uint8_t)(four >> (8 * i));
      }
      if (stored && quarter == 0) to[(size_t)16 * a.page + off] = (uint8_t)byte;
    }
    return;
  }
  // queries
  const int pieces = half / 8, groups = (a.nh + kHeads - 1) / kHeads;
  const long long item = (long long)(blockIdx.x - a.kv_blocks) * 256 + threadIdx.x;
  const int t = (int)(item / (groups * pieces)), rest = (int)(item % (groups * pieces));
  if (t >= a.n) return;
  const int head0 = rest / pieces * kHeads, c = rest % pieces * 8;
  const T* src = (const T*)a.qkv + (size_t)t * a.stride + c;
  T* dst = (T*)a.q + (size_t)t * a.q_stride + c;
  float cs[8], sn[8], x0[kHeads][8], x1[kHeads][8];
  if (a.cosv) {
    load8(a.cosv + (size_t)t * half + c, a.cs_wide, cs);
    load8(a.sinv + (size_t)t * half + c, a.cs_wide, sn);
  }
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {   // (a last group that is not full reads its last head again)
    const T* p = src + (size_t)min(head0 + h, a.nh - 1) * a.hd;
    load8(p, a.wide, x0[h]);
    load8(p + half, a.wide, x1[h]);
  }
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (head0 + h >= a.nh) return;
    if (a.cosv) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float lo = turned_lo(x0[h][i], x1[h][i], cs[i], sn[i]);
        x1[h][i] = turned_hi(x0[h][i], x1[h][i], cs[i], sn[i]);
        x0[h][i] = lo;
      }
    }
    store8(dst + (size_t)(head0 + h) * a.hd, a.q_wide, x0[h]);
    store8(dst + (size_t)(head0 + h) * a.hd + half, a.q_wide, x1[h]);
  }
}

// Rows back from their slots: the lanes of a wave as above.  A lane takes eight channels: a word of a key; of values a byte of eight rows, of
// which it needs one half.
template <typename T>
__global__ __launch_bounds__(256) void fp4_load_kernel(const int32_t* __restrict__ slots, const uint8_t* __restrict__ k_pages,
                                                      const uint8_t* __restrict__ v_pages, T* __restrict__ k, T* __restrict__ v,
                                                      int k_stride, int v_stride, int n, int nkv, int hd, int page, int pages,
                                                      int k_wide, int v_wide) {
  const int nb = hd / kFp4Block, units = 2 * nkv * nb, lane = threadIdx.x % kWave;
  const int wave = blockIdx.x * 4 + threadIdx.x / kWave;
  const int unit = wave % units, t = wave / units * 16 + lane % 16, quarter = lane / 16;
  const int slot = t < n ? slots[t] : -1;
  if (slot < 0 || slot / page >= pages) return;
  const int head = unit / nb % nkv, b = unit % nb, off = slot % page;
  const uint8_t* block = (unit < nkv * nb ? k_pages : v_pages) + (((size_t)(slot / page) * nkv + head) * nb + b) * fp4_block_bytes(page);
  uint32_t word = 0;
  float unit_of;
  if (unit < nkv * nb) {
    word = *reinterpret_cast<const uint32_t*>(block + off * 16 + quarter * 4);
    unit_of = fp4_unit(block[16 * page + fp4_key_scale_place(off)]);
  } else {
    // (byte by byte: words exchanged between four lanes, as the store does it, take 15 us for 6,151 rows of 8 heads of 128, this 12)
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
  // four heads a lane where that leaves four waves to a compute unit
  const bool pairs = hd % 64 == 0;
  const int each = (long long)((n + 15) / 16) * (nkv + (nh + 3) / 4) * (hd / 32) >= 1024 ? 4 : 1;
  const int head_groups = (nkv + each - 1) / each, k_units = head_groups * (pairs ? hd / 64 : hd / 32), v_units = head_groups * (hd / 32);
  const long long waves = slots ? (long long)((n + 15) / 16) * (k_units + v_units) : 0;
  const long long kv = (waves + 3) / 4, items = turns ? (long long)n * ((nh + each - 1) / each) * (hd / 16) : 0, blocks = kv + (items + 255) / 256;
  if (n == 0 || blocks == 0) return 0;
  GB_REQUIRE(blocks < (1ll << 31) && waves < (1ll << 31), "fp4_store: %d rows are too many for one launch", n);
  const StoreArgs a{qkv, q, cosv, sinv, slots, (uint8_t*)k_pages, (uint8_t*)v_pages, stride, q_stride, n, nh, nkv, hd, page, pages,
                    aligned16(qkv) && (size_t)stride * e % 16 == 0, aligned16(q) && (size_t)q_stride * e % 16 == 0,
                    aligned16(cosv) && aligned16(sinv), (int)kv, k_units, v_units};
  const dim3 grid((unsigned)blocks), threads(256);
#define GB_FP4_STORE(T, PAIRS)                                                                                 \
  if (each == 4) hipLaunchKernelGGL((fp4_store_kernel<T, PAIRS, 4>), grid, threads, 0, stream, a);               \
  else hipLaunchKernelGGL((fp4_store_kernel<T, PAIRS, 1>), grid, threads, 0, stream, a);
  if (dtype == kF32 && pairs) { GB_FP4_STORE(float, true) }
  else if (dtype == kF32) { GB_FP4_STORE(float, false) }
  else if (pairs) { GB_FP4_STORE(bf16, true) }
  else { GB_FP4_STORE(bf16, false) }
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
