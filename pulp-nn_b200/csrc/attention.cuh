// attention.cuh -- what the cache kernels (kv_cache.cu) and the attention kernels (attn_decode.cu, attn_prompt.cu)
// share: checks of arguments, the cache as the kernels see it, 16-bit types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <initializer_list>

#include "internal.cuh"

namespace pulpnn {
namespace attn {

constexpr int MAX_HEAD_DIM = 128;

inline int type_size(int type)
{
  switch (type) {
    case PULPNN_TYPE_F16: case PULPNN_TYPE_BF16: return 2;
    case PULPNN_TYPE_F32: case PULPNN_TYPE_S32: return 4;
    case PULPNN_TYPE_S8: case PULPNN_TYPE_U8: return 1;
    default: return 0;
  }
}
inline bool is_wide(int type) { return type == PULPNN_TYPE_F16 || type == PULPNN_TYPE_BF16; }

// records the error and returns its code from the calling function
#define ATTN_REQUIRE(cond, code, ...)       \
  do {                                      \
    if (!(cond)) {                          \
      set_error(code, __VA_ARGS__);         \
      return code;                          \
    }                                       \
  } while (0)

// A kernel that reads a host pointer faults, and one that reads another GPU's memory may: neither is launched. (In kv_cache.cu.)
bool on_device(const Context &c, const char *who, std::initializer_list<const void *> pointers);

inline bool aligned(const void *p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (unsigned)(bytes - 1)) == 0; }
// rows of `size`-byte elements at these strides begin on 16-byte boundaries
inline bool rows_aligned(const void *p, int size, std::initializer_list<int64_t> strides)
{
  if (!aligned(p, 16)) return false;
  for (int64_t s : strides)
    if ((s * size) & 15) return false;
  return true;
}

// rows of an attention's output: stored four channels at a time
inline bool out_aligned(const void *p, int type, int64_t s0, int64_t s1)
{
  const int size = type_size(type);
  return type != PULPNN_TYPE_U8 ? rows_aligned(p, size, {s0, s1}) : aligned(p, 4) && s0 % 4 == 0 && s1 % 4 == 0;
}

int check_cache(const char *who, const pulpnn_kv_cache_t *cache);
inline int check_scale(const char *who, float scale)
{
  ATTN_REQUIRE(scale > 0.f && scale < 1e30f, PULPNN_ERR_INVALID_ARG, "%s: scale %g", who, (double)scale);
  return PULPNN_OK;
}
// step and zero point of a uint8 output
inline int check_out(const char *who, int type, float step, int zero)
{
  ATTN_REQUIRE(type != PULPNN_TYPE_U8 || (step > 1e-30f && step < 1e30f && zero >= 0 && zero <= 255), PULPNN_ERR_INVALID_ARG,
               "%s: uint8 output with step %g and zero point %d", who, (double)step, zero);
  return PULPNN_OK;
}

// The cache as the kernels see it. Slots are below 2^31 (check_cache), so that a slot's page is a 32-bit division.
struct CacheView {
  char *k, *v;
  float *k_scale, *v_scale;
  int64_t page_stride, slot_stride, head_stride;
  int64_t s_page_stride, s_slot_stride, s_head_stride;
  int n_slots, n_pages, page_size, n_heads;
  FastDiv by_page;
};
inline CacheView view_of(const pulpnn_kv_cache_t &c)
{
  CacheView v;
  v.k = static_cast<char *>(c.k); v.v = static_cast<char *>(c.v);
  v.k_scale = c.k_scale; v.v_scale = c.v_scale;
  v.page_stride = c.page_stride; v.slot_stride = c.slot_stride; v.head_stride = c.head_stride;
  v.s_page_stride = c.scale_page_stride; v.s_slot_stride = c.scale_slot_stride; v.s_head_stride = c.scale_head_stride;
  v.n_slots = c.n_pages * c.page_size; v.n_pages = c.n_pages; v.page_size = c.page_size; v.n_heads = c.n_heads;
  v.by_page.set((unsigned)c.page_size);
  return v;
}

#ifdef __CUDACC__
__device__ __forceinline__ int64_t row_of(const CacheView &c, int page, int at, int head)
{
  return page * c.page_stride + at * c.slot_stride + head * c.head_stride;
}
__device__ __forceinline__ int64_t scale_of(const CacheView &c, int page, int at, int head)
{
  return page * c.s_page_stride + at * c.s_slot_stride + head * c.s_head_stride;
}

// two values of a 16-bit type in one word, the first in the low half; rounded to nearest even
template <typename T> __device__ __forceinline__ unsigned pack2(float a, float b);
template <> __device__ __forceinline__ unsigned pack2<__half>(float a, float b)
{
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned *>(&h);
}
template <> __device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float a, float b)
{
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned *>(&h);
}
template <typename T> __device__ __forceinline__ float2 unpack2(unsigned w);
template <> __device__ __forceinline__ float2 unpack2<__half>(unsigned w)
{
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(unsigned w)
{
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// Signed bytes as fp16: a byte plus 128 in the low bits of 1024 is 1152 + code, exactly. `biased` holds bytes ^ 0x80, two of
// which `select` puts into the low bytes of the halves.
__device__ __forceinline__ unsigned widen(unsigned biased, unsigned select)
{
  const unsigned w = __byte_perm(biased, 0x64646464u, select), off = 0x64806480u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&w), *reinterpret_cast<const __half2 *>(&off));
  return *reinterpret_cast<const unsigned *>(&r);
}
// four adjacent channels of an output row; uint8: rint(y * (1 / step)) + zero, cut to 0 .. 255 (a NaN gives the zero point)
__device__ __forceinline__ unsigned to_u8(float y, float inv_step, int zero)
{
  const float x = fminf(fmaxf(y * inv_step, -1e6f), 1e6f);
  return (unsigned)clip_u8((y == y ? __float2int_rn(x) : 0) + zero);
}
__device__ __forceinline__ void store4(char *row, int channel, int type, const float (&y)[4], float inv_step, int zero)
{
  if (type == PULPNN_TYPE_U8)
    *reinterpret_cast<unsigned *>(row + channel) = to_u8(y[0], inv_step, zero) | to_u8(y[1], inv_step, zero) << 8 |
                                                   to_u8(y[2], inv_step, zero) << 16 | to_u8(y[3], inv_step, zero) << 24;
  else if (type == PULPNN_TYPE_F16)
    *reinterpret_cast<uint2 *>(row + channel * 2) = make_uint2(pack2<__half>(y[0], y[1]), pack2<__half>(y[2], y[3]));
  else
    *reinterpret_cast<uint2 *>(row + channel * 2) = make_uint2(pack2<__nv_bfloat16>(y[0], y[1]), pack2<__nv_bfloat16>(y[2], y[3]));
}
#endif

}  // namespace attn
}  // namespace pulpnn
