// kv_cache.cu -- rows into and out of a paged cache of keys and values: pulpnn_kv_append (position rotation of
// queries and keys, storing with a cut to 8 bits) and pulpnn_kv_gather.
//
// Both move bytes: 48 rows of 128 channels a token at 32 query and 8 key heads, some 4 operations a channel. A warp of the
// append holds whole rows, as many as fit at 16 or 8 channels a lane (6 or 3 of 80 channels), so that it loads and stores them in
// 16-byte pieces and a row's largest value is 3 or 4 shuffles away.
//
// Measured (one B200; the copy rate is 6.56 TB/s): 32-bit accumulators of 4096 tokens, 32 query and 8 key heads of 128 channels,
// into an 8-bit cache and 16-bit queries, 30.6 us (4.7 TB/s; of 32768 tokens 197 us, 5.8 TB/s); 32768 tokens of 16 heads of 80
// channels in 16 bits, 32 of them rotated, 80 us (6.3 TB/s); 8 tokens 2.2 us. The gather of 100003 tokens of 8 heads of 128
// channels out of 8 bits 107 us (5.8 TB/s).
#include <cuda.h>

#include "attention.cuh"

namespace pulpnn {
namespace attn {

typedef CUresult (*PointerAttributeFn)(void *, CUpointer_attribute, CUdeviceptr);

bool on_device(const Context &c, const char *who, std::initializer_list<const void *> pointers)
{
  // one attribute of the driver's takes half the time of the runtime's whole answer, and a call has up to thirteen pointers
  static PointerAttributeFn attribute = [] {
    void *f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuPointerGetAttribute", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<PointerAttributeFn>(f);
  }();
  static const int devices = [] {
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess) cudaGetLastError();
    return n;
  }();
  for (const void *p : pointers) {
    if (!p) continue;
    unsigned type = 0;
    int device = c.device;
    const CUdeviceptr at = reinterpret_cast<CUdeviceptr>(p);
    if (attribute && attribute(&type, CU_POINTER_ATTRIBUTE_MEMORY_TYPE, at) == CUDA_SUCCESS && type == CU_MEMORYTYPE_DEVICE &&
        (devices == 1 || (attribute(&device, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL, at) == CUDA_SUCCESS && device == c.device)))
      continue;
    cudaPointerAttributes a;
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
      cudaGetLastError();
      set_error(PULPNN_ERR_INVALID_ARG, "%s: %p is not an address CUDA knows", who, p);
      return false;
    }
    if (a.type == cudaMemoryTypeManaged) continue;
    if (a.type != cudaMemoryTypeDevice || a.device != c.device) {
      set_error(PULPNN_ERR_INVALID_ARG, "%s: %p is not memory of GPU %d", who, p, c.device);
      return false;
    }
  }
  return true;
}

int check_cache(const char *who, const pulpnn_kv_cache_t *c)
{
  ATTN_REQUIRE(c && c->k && c->v, PULPNN_ERR_INVALID_ARG, "%s: no cache", who);
  ATTN_REQUIRE(is_wide(c->type) || c->type == PULPNN_TYPE_S8, PULPNN_ERR_INVALID_ARG, "%s: cache type %d", who, c->type);
  const bool eight = c->type == PULPNN_TYPE_S8;
  ATTN_REQUIRE(!eight || (c->k_scale && c->v_scale), PULPNN_ERR_INVALID_ARG, "%s: an 8-bit cache without scales", who);
  ATTN_REQUIRE(c->n_pages > 0 && c->page_size > 0 && c->n_heads > 0, PULPNN_ERR_INVALID_ARG,
               "%s: a cache of %d pages, %d slots, %d heads", who, c->n_pages, c->page_size, c->n_heads);
  ATTN_REQUIRE((int64_t)c->n_pages * c->page_size <= 0x7fffffff, PULPNN_ERR_UNSUPPORTED, "%s: a cache of 2^31 slots or more", who);
  ATTN_REQUIRE(c->n_heads <= 65535, PULPNN_ERR_UNSUPPORTED, "%s: %d heads", who, c->n_heads);
  const int unit = eight ? 16 : 8;
  ATTN_REQUIRE(c->head_dim > 0 && c->head_dim <= MAX_HEAD_DIM && c->head_dim % unit == 0, PULPNN_ERR_UNSUPPORTED,
               "%s: head_dim %d is not a multiple of %d up to %d", who, c->head_dim, unit, MAX_HEAD_DIM);
  const int size = type_size(c->type);
  ATTN_REQUIRE(rows_aligned(c->k, size, {c->page_stride, c->slot_stride, c->head_stride}) && aligned(c->v, 16),
               PULPNN_ERR_UNSUPPORTED, "%s: the cache's rows do not begin on 16-byte boundaries", who);
  ATTN_REQUIRE(!eight || (aligned(c->k_scale, 4) && aligned(c->v_scale, 4)), PULPNN_ERR_INVALID_ARG, "%s: unaligned scales", who);
  return PULPNN_OK;
}

namespace {

constexpr int THREADS = 256;               // of a gather's block
constexpr int WARPS = 4, MOST_TOKENS = 8;  // of an append's

struct AppendProblem {
  const char *in[3];          // q, k, v
  char *out[3];
  const float *step[3];
  int step_vector[3];         // begins on a 16-byte boundary
  int64_t in_token[3], in_head[3], out_token[3], out_head[3];      // bytes
  const long long *slots;
  const int *positions;
  const double *inv_freq;
  CacheView cache;
  int n, heads[3], tokens[3], blocks[3];                 // of q, k, v: heads; tokens of a block; blocks
  FastDiv by_heads[3];
  int dim, half, interleaved, chunks, pow2, narrow, per_warp;                       // chunks of a row, one a lane; rows of a warp
};

struct S32 {};
struct F32 {};

// four channels as they come
template <typename IN> struct Raw { uint2 v; };
template <> struct Raw<S32> { uint4 v; };
template <> struct Raw<F32> { uint4 v; };
template <typename IN> struct Width { static constexpr int v = sizeof(Raw<IN>) / 4; };

template <typename IN> __device__ __forceinline__ Raw<IN> load4(const char *p) { return *reinterpret_cast<const Raw<IN> *>(p); }
template <typename IN> __device__ __forceinline__ void values(const Raw<IN> &w, float *x)
{
  const float2 a = unpack2<IN>(w.v.x), b = unpack2<IN>(w.v.y);
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}
template <> __device__ __forceinline__ void values<S32>(const Raw<S32> &w, float *x)
{
  x[0] = (float)(int)w.v.x; x[1] = (float)(int)w.v.y; x[2] = (float)(int)w.v.z; x[3] = (float)(int)w.v.w;
}
template <> __device__ __forceinline__ void values<F32>(const Raw<F32> &w, float *x)
{
  x[0] = __uint_as_float(w.v.x); x[1] = __uint_as_float(w.v.y); x[2] = __uint_as_float(w.v.z); x[3] = __uint_as_float(w.v.w);
}
template <typename IN> __device__ __forceinline__ float load1(const char *p) { return (float)*reinterpret_cast<const IN *>(p); }
template <> __device__ __forceinline__ float load1<S32>(const char *p) { return (float)*reinterpret_cast<const int *>(p); }
template <> __device__ __forceinline__ float load1<F32>(const char *p) { return *reinterpret_cast<const float *>(p); }
// times the real value of a step, channel by channel
__device__ __forceinline__ void times4(const float *step, bool vector, float *x)
{
  if (vector) {
    const float4 s = __ldg(reinterpret_cast<const float4 *>(step));
    x[0] *= s.x; x[1] *= s.y; x[2] *= s.z; x[3] *= s.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] *= __ldg(step + i);
  }
}
// the larger magnitude; NaN where one of them is
__device__ __forceinline__ float larger(float a, float b)
{
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}
// x * inv to the nearest integer, ties to even, in the low byte: 1.5 * 2^23 leaves the sum no bits below one. inv = (1 / most) * 127 is
// rounded twice, so that next to a tie (127 * 1.5 * 2^-23, below 2^-15) the neighbour may come out; a division a value would cost more
// than all the rest.
__device__ __forceinline__ unsigned code(float x, float inv) { return __float_as_uint(fmaf(x, inv, 12582912.f)); }

// One block: the queries, the keys or the values of a few tokens, as many as give each thread about BATCH rows, so that
// strides and addresses are the whole block's, and the tokens' angles and slots are looked up once. A warp holds per_warp whole
// rows; BATCH loads of a thread are under way together, the first of them while the angles are computed.
// A lane has OCTS times eight channels of a row. HALVES (all channels rotate, or none): eight are four of each half of the row, so
// that it has both of every pair, whichever way they are paired, and 32-bit rows are read without gaps between the lanes. Otherwise
// eight side by side, whose mates come from another lane, or one by one where they are not eight side by side either.
// NARROW: what a block's rows lie apart fits 32 bits, as it nearly always does; products of 64 bits were a fifth of the instructions.
template <bool NARROW> __device__ __forceinline__ int64_t apart(int a, int64_t sa, int b, int64_t sb)
{
  return NARROW ? (int64_t)(a * (int)sa + b * (int)sb) : a * sa + b * sb;
}
constexpr int64_t NOWHERE = INT64_MIN;       // no place is that; others may be below zero, where strides are
// What the cache holds: the outputs' type, the other 16-bit type, or 8 bits.
enum Held { SAME, OTHER, CODES };
template <typename T> struct OtherType { typedef __half type; };
template <> struct OtherType<__half> { typedef __nv_bfloat16 type; };
template <typename IN, typename WIDE, Held HELD, bool HALVES, bool NARROW, int OCTS>
__global__ void __launch_bounds__(WARPS * 32, Width<IN>::v == 2 ? 10 : 8) kv_append_kernel(const AppendProblem p)
{
  constexpr int SIZE = Width<IN>::v, BATCH = (SIZE == 2 ? 4 : 2) / OCTS;
  __shared__ __align__(16) float2 turns[MOST_TOKENS][MAX_HEAD_DIM / 2];
  __shared__ longlong2 where[MOST_TOKENS];      // of a token's head 0: its row's and its scale's place in the cache; NOWHERE: it is not stored
  const int which = blockIdx.x < p.blocks[0] ? 0 : (blockIdx.x < p.blocks[0] + p.blocks[1] ? 1 : 2);
  const int block = blockIdx.x - (which > 0 ? p.blocks[0] : 0) - (which > 1 ? p.blocks[1] : 0);
  const int token0 = block * p.tokens[which], tokens = min(p.tokens[which], p.n - token0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / p.chunks, chunk = lane - sub * p.chunks, first_lane = sub * p.chunks;
  int c0[OCTS], c1[OCTS];        // two times four channels of each of its octets
#pragma unroll
  for (int o = 0; o < OCTS; o++) {
    c0[o] = (o * p.chunks + chunk) * (HALVES ? 4 : 8);
    c1[o] = HALVES ? p.dim / 2 + c0[o] : c0[o] + 4;
  }
  const int heads = p.heads[which], rows = tokens * heads, half = which < 2 ? p.half : 0;
  const FastDiv by_heads = p.by_heads[which];
  const int64_t in_head = p.in_head[which], out_head = p.out_head[which], in_token = p.in_token[which], out_token = p.out_token[which];
  const char *in = p.in[which] + token0 * in_token;
  char *out = p.out[which] ? p.out[which] + token0 * out_token : nullptr;
  const float *steps = sizeof(IN) == 1 ? p.step[which] : nullptr;       // of S32 only
  char *held = which == 1 ? p.cache.k : p.cache.v;
  const int stride = WARPS * p.per_warp;
  pdl_wait();
  for (int base = 0; base < rows; base += BATCH * stride) {
    Raw<IN> lo[BATCH][OCTS], hi[BATCH][OCTS];
    int head[BATCH], token[BATCH];
    bool live[BATCH];
#pragma unroll
    for (int b = 0; b < BATCH; b++) {
      const int row = base + b * stride + warp * p.per_warp + sub;
      live[b] = sub < p.per_warp && row < rows;
      token[b] = by_heads.div(row); head[b] = row - token[b] * heads;
      if (live[b]) {
        const char *src = in + apart<NARROW>(token[b], in_token, head[b], in_head);
#pragma unroll
        for (int o = 0; o < OCTS; o++) {
          if (!HALVES && SIZE == 2) {
            const uint4 both = *reinterpret_cast<const uint4 *>(src + c0[o] * SIZE);
            reinterpret_cast<uint2 &>(lo[b][o]) = make_uint2(both.x, both.y); reinterpret_cast<uint2 &>(hi[b][o]) = make_uint2(both.z, both.w);
          } else {
            lo[b][o] = load4<IN>(src + c0[o] * SIZE); hi[b][o] = load4<IN>(src + c1[o] * SIZE);
          }
        }
      }
    }
    if (base == 0) {
      for (int i = threadIdx.x; i < tokens * half; i += WARPS * 32) {
        // The angle in turns, in 64 bits: a position of 10^5 times a frequency near 1 leaves 32 bits with errors of 10^-2.
        // Its fraction of a turn keeps 24 bits, and sincospif takes multiples of pi.
        const int k = i / half, f = i - k * half;
        const double t = (double)__ldg(p.positions + token0 + k) * __ldg(p.inv_freq + f) * 0.15915494309189533577;
        float s, c;
        sincospif(2.f * (float)(t - rint(t)), &s, &c);
        turns[k][f] = make_float2(c, s);
      }
      if (which && threadIdx.x < tokens) {
        const long long slot = __ldg(p.slots + token0 + threadIdx.x);
        const bool stored = slot >= 0 && slot < p.cache.n_slots;
        const int page = stored ? p.cache.by_page.div((int)slot) : 0, at = stored ? (int)slot - page * p.cache.page_size : 0;
        where[threadIdx.x] = stored ? make_longlong2(row_of(p.cache, page, at, 0), scale_of(p.cache, page, at, 0)) : make_longlong2(NOWHERE, 0);
      }
      __syncthreads();
    }
#pragma unroll
    for (int b = 0; b < BATCH; b++) {
      if (!__any_sync(0xffffffffu, live[b])) break;
      const int k = live[b] ? token[b] : 0;
      const float2 *turn = turns[k];
      float y[OCTS][8];
      uint2 wide0[OCTS], wide1[OCTS];
#pragma unroll
      for (int o = 0; o < OCTS; o++) {
        float x[8];
        if (!live[b]) lo[b][o] = hi[b][o] = Raw<IN>{};
        values<IN>(lo[b][o], x);
        values<IN>(hi[b][o], x + 4);
        if (sizeof(IN) == 1 && steps && live[b]) {
          times4(steps + head[b] * p.dim + c0[o], p.step_vector[which], x);
          times4(steps + head[b] * p.dim + c1[o], p.step_vector[which], x + 4);
        }
        float *const w = y[o];
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = x[i];
        if (HALVES && half && !p.interleaved) {
          const float4 u = *reinterpret_cast<const float4 *>(turn + c0[o]), v = *reinterpret_cast<const float4 *>(turn + c0[o] + 2);
          const float cs[4] = {u.x, u.z, v.x, v.z}, sn[4] = {u.y, u.w, v.y, v.w};
#pragma unroll
          for (int i = 0; i < 4; i++) {
            w[i] = x[i] * cs[i] - x[i + 4] * sn[i];
            w[i + 4] = x[i + 4] * cs[i] + x[i] * sn[i];
          }
        } else if (half && p.interleaved) {
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            const int c = i == 0 ? c0[o] : c1[o];
            if (c < 2 * half) {
              float4 u = *reinterpret_cast<const float4 *>(turn + (c >> 1));
              if (c + 2 >= 2 * half) { u.z = 1.f; u.w = 0.f; }
              w[i] = x[i] * u.x - x[i + 1] * u.y; w[i + 1] = x[i + 1] * u.x + x[i] * u.y;
              w[i + 2] = x[i + 2] * u.z - x[i + 3] * u.w; w[i + 3] = x[i + 3] * u.z + x[i + 2] * u.w;
            }
          }
        } else if (OCTS == 1 && !HALVES && half && (half & 7) == 0) {
          const bool low = c0[o] < half;
          const int mate = (lane + (low ? half >> 3 : -(half >> 3))) & 31;
          float z[8];
#pragma unroll
          for (int i = 0; i < 8; i++) z[i] = __shfl_sync(0xffffffffu, x[i], mate);
          if (c0[o] < 2 * half) {
            const float sign = low ? -1.f : 1.f;
            const float4 *t = reinterpret_cast<const float4 *>(turn + (low ? c0[o] : c0[o] - half));
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
              const float4 u = t[i / 2];
              w[i] = x[i] * u.x + z[i] * (sign * u.y);
              w[i + 1] = x[i + 1] * u.z + z[i + 1] * (sign * u.w);
            }
          }
        } else if (OCTS == 1 && !HALVES && half) {
          const char *src = in + token[b] * in_token + head[b] * in_head;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int c = c0[o] + i;
            if (c < 2 * half && live[b]) {
              const bool lower = c < half;
              const int other = lower ? c + half : c - half;
              float z = load1<IN>(src + other * SIZE);
              if (sizeof(IN) == 1 && steps) z *= __ldg(steps + head[b] * p.dim + other);
              const float2 t = turn[lower ? c : other];
              w[i] = x[i] * t.x + (lower ? -z : z) * t.y;
            }
          }
          __syncwarp();          // in place: every lane of the row has read what another lane now writes over
        }
        wide0[o] = make_uint2(pack2<WIDE>(y[o][0], y[o][1]), pack2<WIDE>(y[o][2], y[o][3]));
        wide1[o] = make_uint2(pack2<WIDE>(y[o][4], y[o][5]), pack2<WIDE>(y[o][6], y[o][7]));
      }
      auto put = [&](char *row) {
#pragma unroll
        for (int o = 0; o < OCTS; o++) {
          if (HALVES) {
            *reinterpret_cast<uint2 *>(row + c0[o] * 2) = wide0[o];
            *reinterpret_cast<uint2 *>(row + c1[o] * 2) = wide1[o];
          } else {
            *reinterpret_cast<uint4 *>(row + c0[o] * 2) = make_uint4(wide0[o].x, wide0[o].y, wide1[o].x, wide1[o].y);
          }
        }
      };
      if (live[b] && out) put(out + apart<NARROW>(token[b], out_token, head[b], out_head));
      if (which == 0) continue;
      const longlong2 at = where[k];
      const bool stored = live[b] && at.x != NOWHERE;
      const int64_t place = at.x + apart<NARROW>(head[b], p.cache.head_stride, 0, 0);
      if (HELD == CODES) {
        float most = 0.f;
#pragma unroll
        for (int o = 0; o < OCTS; o++)
#pragma unroll
          for (int i = 0; i < 8; i++) most = larger(most, y[o][i]);
        if (p.pow2) {
#pragma unroll
          for (int d = 1; d < 16; d *= 2)
            if (d < p.chunks) most = larger(most, __shfl_xor_sync(0xffffffffu, most, d));
        } else {
          // around the row's lanes: after steps of 1, 2, 4 and 8 each of up to 16 has met all others
#pragma unroll
          for (int d = 1; d < 16; d *= 2) {
            int from = lane - first_lane + d;
            while (from >= p.chunks) from -= p.chunks;
            most = larger(most, __shfl_sync(0xffffffffu, most, (first_lane + from) & 31));
          }
        }
        if (stored) {
          const bool fine = most <= 3.402823466e38f, any = most >= 7.888609e-31f && fine;     // 2^-100
          const float inv = __frcp_rn(most) * 127.f;
          char *row = held + place;
#pragma unroll
          for (int o = 0; o < OCTS; o++) {
            const float *z = y[o];
            unsigned w0 = 0, w1 = 0;
            if (any) {
              w0 = __byte_perm(__byte_perm(code(z[0], inv), code(z[1], inv), 0x0040), __byte_perm(code(z[2], inv), code(z[3], inv), 0x0040), 0x5410);
              w1 = __byte_perm(__byte_perm(code(z[4], inv), code(z[5], inv), 0x0040), __byte_perm(code(z[6], inv), code(z[7], inv), 0x0040), 0x5410);
            }
            *reinterpret_cast<unsigned *>(row + c0[o]) = w0;
            *reinterpret_cast<unsigned *>(row + c1[o]) = w1;
          }
          if (chunk == 0)
            (which == 1 ? p.cache.k_scale : p.cache.v_scale)[at.y + head[b] * p.cache.s_head_stride] =
                any ? most * (1.f / 127.f) : (fine ? 0.f : __int_as_float(0x7fffffff));
        }
      } else if (stored) {
        if (HELD == OTHER) {
          typedef typename OtherType<WIDE>::type O;
#pragma unroll
          for (int o = 0; o < OCTS; o++) {
            const float *z = y[o];
            wide0[o] = make_uint2(pack2<O>(z[0], z[1]), pack2<O>(z[2], z[3])); wide1[o] = make_uint2(pack2<O>(z[4], z[5]), pack2<O>(z[6], z[7]));
          }
        }
        put(held + place * 2);
      }
    }
  }
}

template <typename IN, typename WIDE, Held HELD>
cudaError_t append_go(AppendProblem &p, int sms, cudaStream_t s)
{
  // Two octets of channels a lane where no lane needs another's channels: a row's index, addresses and maximum are shared by twice
  // as many (accumulators of 4096 tokens into 8 bits 30.6 us, with one octet 31.7; 32768 tokens of 80 channels in 16 bits 80, 87).
  const bool halves = p.half == 0 || 2 * p.half == p.dim;
  const bool two = p.dim % 16 == 0 && p.narrow && (halves || p.interleaved);
  p.chunks = p.dim / (two ? 16 : 8); p.pow2 = (p.chunks & (p.chunks - 1)) == 0; p.per_warp = 32 / p.chunks;
  // Tokens of a block: for eight octets a thread where there are blocks enough, else one (four of 16-bit rows: 5 % slower; two of 32-bit
  // ones: 4 %).
  const int rows = WARPS * p.per_warp * (two ? 4 : 8);
  unsigned blocks = 0;
  for (int i = 0; i < 3; i++) {
    p.tokens[i] = 1; p.blocks[i] = 0;
    if (p.heads[i] == 0) continue;
    while (p.tokens[i] < MOST_TOKENS && p.tokens[i] * p.heads[i] < rows && p.n >= 4 * sms * (p.tokens[i] + 1)) p.tokens[i]++;
    p.by_heads[i].set((unsigned)p.heads[i]);
    p.blocks[i] = (p.n + p.tokens[i] - 1) / p.tokens[i];
    blocks += (unsigned)p.blocks[i];
  }
  auto k = two ? (halves ? kv_append_kernel<IN, WIDE, HELD, true, true, 2> : kv_append_kernel<IN, WIDE, HELD, false, true, 2>)
               : (p.narrow ? (halves ? kv_append_kernel<IN, WIDE, HELD, true, true, 1> : kv_append_kernel<IN, WIDE, HELD, false, true, 1>)
                           : (halves ? kv_append_kernel<IN, WIDE, HELD, true, false, 1> : kv_append_kernel<IN, WIDE, HELD, false, false, 1>));
  return launch_pdl(k, dim3(blocks), dim3(WARPS * 32), 0, s, p);
}
template <typename WIDE, Held HELD>
cudaError_t append_in(int in_type, AppendProblem &p, int sms, cudaStream_t s)
{
  switch (in_type) {
    case PULPNN_TYPE_F16: return append_go<__half, WIDE, HELD>(p, sms, s);
    case PULPNN_TYPE_BF16: return append_go<__nv_bfloat16, WIDE, HELD>(p, sms, s);
    case PULPNN_TYPE_F32: return append_go<F32, WIDE, HELD>(p, sms, s);
    default: return append_go<S32, WIDE, HELD>(p, sms, s);
  }
}

template <typename WIDE>
cudaError_t append_held(Held held, int in_type, AppendProblem &p, int sms, cudaStream_t s)
{
  return held == CODES ? append_in<WIDE, CODES>(in_type, p, sms, s)
                       : (held == SAME ? append_in<WIDE, SAME>(in_type, p, sms, s) : append_in<WIDE, OTHER>(in_type, p, sms, s));
}

struct GatherProblem {
  const long long *slots;
  char *out[2];
  int64_t out_token[2], out_head[2];      // bytes
  CacheView cache;
  int n, dim, chunks, per_block, heads, whole;   // chunks of 16 bytes in a cached row; rows of a block at a time
  FastDiv by_heads;
};

// Rows (token, head), heads fastest, a chunk of 16 cached bytes a thread; blockIdx.y is keys or values. A thread takes BATCH
// rows, a block's rows apart, and has all their loads under way before it stores the first.
template <typename WIDE, bool EIGHT>
__global__ void __launch_bounds__(THREADS) kv_gather_kernel(const GatherProblem p)
{
  constexpr int BATCH = 2;                 // of 100003 rows of 8 heads: 106 us; one 114, four 114
  const int sub = threadIdx.x / p.chunks, chunk = threadIdx.x - sub * p.chunks, which = p.out[0] ? blockIdx.y : 1;
  const char *from = which == 0 ? p.cache.k : p.cache.v;
  const float *scales = which == 0 ? p.cache.k_scale : p.cache.v_scale;
  pdl_wait();
  if (sub >= p.per_block) return;
  uint4 w[BATCH];
  float scale[BATCH];
  int64_t to[BATCH];
#pragma unroll
  for (int b = 0; b < BATCH; b++) {
    const int row = (blockIdx.x * BATCH + b) * p.per_block + sub;
    to[b] = NOWHERE;
    w[b] = make_uint4(0, 0, 0, 0);
    scale[b] = 0.f;
    const int token = p.by_heads.div(row), head = row - token * p.heads;
    if (token >= p.n) continue;
    to[b] = token * p.out_token[which] + head * p.out_head[which] + chunk * (EIGHT ? 32 : 16);
    const long long slot = __ldg(p.slots + token);
    if (slot < 0 || slot >= p.cache.n_slots) continue;
    const int page = p.cache.by_page.div((int)slot), at = (int)slot - page * p.cache.page_size;
    w[b] = *reinterpret_cast<const uint4 *>(from + row_of(p.cache, page, at, head) * (EIGHT ? 1 : 2) + chunk * 16);
    if (EIGHT) scale[b] = scales[scale_of(p.cache, page, at, head)];
  }
#pragma unroll
  for (int b = 0; b < BATCH; b++) {
    if (to[b] == NOWHERE) continue;
    uint4 *dst = reinterpret_cast<uint4 *>(p.out[which] + to[b]);
    if (!EIGHT) { *dst = w[b]; continue; }
    const unsigned q[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
    unsigned y[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const unsigned u = q[i] ^ 0x80808080u;
      const float2 a = unpack2<__half>(widen(u, 0x4140)), c = unpack2<__half>(widen(u, 0x4342));
      y[2 * i] = pack2<WIDE>(a.x * scale[b], a.y * scale[b]);
      y[2 * i + 1] = pack2<WIDE>(c.x * scale[b], c.y * scale[b]);
    }
    if (p.whole) {       // a full 32-byte sector per lane and instruction
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]), "r"(y[4]),
                   "r"(y[5]), "r"(y[6]), "r"(y[7]) : "memory");
    } else {
      dst[0] = make_uint4(y[0], y[1], y[2], y[3]);
      dst[1] = make_uint4(y[4], y[5], y[6], y[7]);
    }
  }
}

template <typename WIDE, bool EIGHT>
cudaError_t gather_go(GatherProblem &p, cudaStream_t s)
{
  p.chunks = p.dim * (EIGHT ? 1 : 2) / 16; p.per_block = THREADS / p.chunks; p.heads = p.cache.n_heads;
  p.by_heads.set((unsigned)p.heads);
  p.whole = 1;
  for (int i = 0; i < 2; i++)
    if (p.out[i] && (!aligned(p.out[i], 32) || p.out_token[i] % 32 || p.out_head[i] % 32)) p.whole = 0;
  const int64_t rows = (int64_t)p.n * p.heads, per = 2 * p.per_block;
  const dim3 grid((unsigned)((rows + per - 1) / per), p.out[0] && p.out[1] ? 2 : 1);
  return launch_pdl(kv_gather_kernel<WIDE, EIGHT>, grid, dim3(THREADS), 0, s, p);
}

}  // namespace
}  // namespace attn
}  // namespace pulpnn

using namespace pulpnn;
using namespace pulpnn::attn;

extern "C" int pulpnn_kv_append(const pulpnn_kv_cache_t *cache, const pulpnn_kv_append_t *a)
{
  const char *who = "pulpnn_kv_append";
  Context &c = ctx();
  if (const int e = check_cache(who, cache)) return e;
  ATTN_REQUIRE(a && a->n_tokens >= 0, PULPNN_ERR_INVALID_ARG, "%s: %d tokens", who, a ? a->n_tokens : -1);
  if (a->n_tokens == 0) return PULPNN_OK;
  ATTN_REQUIRE(a->k && a->v && a->slots, PULPNN_ERR_INVALID_ARG, "%s: NULL pointer", who);
  ATTN_REQUIRE(is_wide(a->out_type), PULPNN_ERR_INVALID_ARG, "%s: out_type %d", who, a->out_type);
  ATTN_REQUIRE(is_wide(a->in_type) || a->in_type == PULPNN_TYPE_F32 || a->in_type == PULPNN_TYPE_S32, PULPNN_ERR_INVALID_ARG,
               "%s: in_type %d", who, a->in_type);
  ATTN_REQUIRE((a->q != nullptr) == (a->q_out != nullptr), PULPNN_ERR_INVALID_ARG, "%s: q without q_out, or q_out without q", who);
  ATTN_REQUIRE(!a->q || (a->n_q_heads > 0 && a->n_q_heads <= 65535), PULPNN_ERR_INVALID_ARG, "%s: %d query heads", who, a->n_q_heads);
  ATTN_REQUIRE(a->n_tokens <= 0x2aaaaaaa, PULPNN_ERR_UNSUPPORTED, "%s: %d tokens", who, a->n_tokens);
  ATTN_REQUIRE(a->rotary_dim >= 0 && a->rotary_dim <= cache->head_dim && a->rotary_dim % 2 == 0, PULPNN_ERR_INVALID_ARG,
               "%s: rotary_dim %d of %d channels", who, a->rotary_dim, cache->head_dim);
  ATTN_REQUIRE(a->rotary_dim == 0 || (a->positions && a->inv_freq), PULPNN_ERR_INVALID_ARG, "%s: a rotation without positions or frequencies", who);
  const bool s32 = a->in_type == PULPNN_TYPE_S32;
  ATTN_REQUIRE(!s32 || ((a->q_step || !a->q) && a->k_step && a->v_step), PULPNN_ERR_INVALID_ARG, "%s: S32 input without steps", who);
  const int is = type_size(a->in_type);
  ATTN_REQUIRE((!a->q || (rows_aligned(a->q, is, {a->q_stride[0], a->q_stride[1]}) &&
                          rows_aligned(a->q_out, 2, {a->q_out_stride[0], a->q_out_stride[1]}))) &&
               rows_aligned(a->k, is, {a->k_stride[0], a->k_stride[1]}) && rows_aligned(a->v, is, {a->v_stride[0], a->v_stride[1]}) &&
               (!a->k_out || rows_aligned(a->k_out, 2, {a->k_out_stride[0], a->k_out_stride[1]})) &&
               (!a->v_out || rows_aligned(a->v_out, 2, {a->v_out_stride[0], a->v_out_stride[1]})),
               PULPNN_ERR_UNSUPPORTED, "%s: rows that do not begin on 16-byte boundaries", who);
  ATTN_REQUIRE(aligned(a->slots, 8) && aligned(a->positions, 4) && aligned(a->inv_freq, 8) && aligned(a->q_step, 4) &&
               aligned(a->k_step, 4) && aligned(a->v_step, 4), PULPNN_ERR_INVALID_ARG, "%s: unaligned slots, positions, frequencies or steps", who);
  if (!ensure_device(c)) return c.err;
  if (!on_device(c, who, {cache->k, cache->v, cache->k_scale, cache->v_scale, a->q, a->k, a->v, a->q_out, a->k_out, a->v_out, a->q_step,
                          a->k_step, a->v_step, a->slots, a->positions, a->inv_freq})) return c.err;

  AppendProblem p;
  const void *in[3] = {a->q, a->k, a->v};
  void *out[3] = {a->q_out, a->k_out, a->v_out};
  const float *step[3] = {a->q_step, a->k_step, a->v_step};
  const int64_t *is_[3] = {a->q_stride, a->k_stride, a->v_stride}, *os[3] = {a->q_out_stride, a->k_out_stride, a->v_out_stride};
  for (int i = 0; i < 3; i++) {
    p.in[i] = static_cast<const char *>(in[i]); p.out[i] = static_cast<char *>(out[i]); p.step[i] = s32 ? step[i] : nullptr; p.step_vector[i] = aligned(step[i], 16);
    p.in_token[i] = is_[i][0] * is; p.in_head[i] = is_[i][1] * is;
    p.out_token[i] = os[i][0] * 2; p.out_head[i] = os[i][1] * 2;
  }
  p.slots = reinterpret_cast<const long long *>(a->slots); p.positions = a->positions; p.inv_freq = a->inv_freq;
  p.cache = view_of(*cache);
  p.n = a->n_tokens; p.heads[0] = a->q ? a->n_q_heads : 0; p.heads[1] = p.heads[2] = cache->n_heads; p.dim = cache->head_dim;
  p.half = a->rotary_dim / 2; p.interleaved = a->interleaved != 0;
  // the furthest apart that rows of a block can be
  auto near = [](int64_t token, int64_t head, int heads) {
    auto size = [](int64_t x) { return (double)(x < 0 ? -x : x); };
    return size(token) * MOST_TOKENS + size(head) * heads < 2147483647.0;
  };
  p.narrow = near(0, cache->head_stride, cache->n_heads);
  for (int i = 0; i < 3; i++)
    p.narrow = p.narrow && near(p.in_token[i], p.in_head[i], p.heads[i]) && (!p.out[i] || near(p.out_token[i], p.out_head[i], p.heads[i]));
  const Held held = cache->type == PULPNN_TYPE_S8 ? CODES : (cache->type == a->out_type ? SAME : OTHER);
  const cudaError_t e = a->out_type == PULPNN_TYPE_F16 ? append_held<__half>(held, a->in_type, p, c.sm_count, c.stream)
                                                       : append_held<__nv_bfloat16>(held, a->in_type, p, c.sm_count, c.stream);
  if (!cuda_ok(e, who)) return c.err;
  count_launch("kv_append_kernel");
  return PULPNN_OK;
}

extern "C" int pulpnn_kv_gather(const pulpnn_kv_cache_t *cache, const pulpnn_kv_gather_t *a)
{
  const char *who = "pulpnn_kv_gather";
  Context &c = ctx();
  if (const int e = check_cache(who, cache)) return e;
  ATTN_REQUIRE(a && a->n_tokens >= 0, PULPNN_ERR_INVALID_ARG, "%s: %d tokens", who, a ? a->n_tokens : -1);
  if (a->n_tokens == 0) return PULPNN_OK;
  ATTN_REQUIRE(a->slots && (a->k_out || a->v_out), PULPNN_ERR_INVALID_ARG, "%s: NULL pointer", who);
  ATTN_REQUIRE(is_wide(a->out_type), PULPNN_ERR_INVALID_ARG, "%s: out_type %d", who, a->out_type);
  ATTN_REQUIRE(cache->type == PULPNN_TYPE_S8 || cache->type == a->out_type, PULPNN_ERR_UNSUPPORTED,
               "%s: a 16-bit cache of another type than out_type", who);
  ATTN_REQUIRE((!a->k_out || rows_aligned(a->k_out, 2, {a->k_out_stride[0], a->k_out_stride[1]})) &&
               (!a->v_out || rows_aligned(a->v_out, 2, {a->v_out_stride[0], a->v_out_stride[1]})),
               PULPNN_ERR_UNSUPPORTED, "%s: rows that do not begin on 16-byte boundaries", who);
  ATTN_REQUIRE(aligned(a->slots, 8), PULPNN_ERR_INVALID_ARG, "%s: unaligned slots", who);
  // rows are counted in 32 bits, up to a block's rows beyond the last
  ATTN_REQUIRE((int64_t)a->n_tokens * cache->n_heads <= 0x7fffffff - 4 * THREADS, PULPNN_ERR_UNSUPPORTED, "%s: %d tokens of %d heads", who, a->n_tokens, cache->n_heads);
  if (!ensure_device(c)) return c.err;
  if (!on_device(c, who, {cache->k, cache->v, cache->k_scale, cache->v_scale, a->slots, a->k_out, a->v_out})) return c.err;

  GatherProblem p;
  p.slots = reinterpret_cast<const long long *>(a->slots);
  p.out[0] = static_cast<char *>(a->k_out); p.out[1] = static_cast<char *>(a->v_out);
  p.out_token[0] = a->k_out_stride[0] * 2; p.out_head[0] = a->k_out_stride[1] * 2;
  p.out_token[1] = a->v_out_stride[0] * 2; p.out_head[1] = a->v_out_stride[1] * 2;
  p.cache = view_of(*cache);
  p.n = a->n_tokens; p.dim = cache->head_dim;
  const bool f16 = a->out_type == PULPNN_TYPE_F16;
  const cudaError_t e = cache->type == PULPNN_TYPE_S8 ? (f16 ? gather_go<__half, true>(p, c.stream) : gather_go<__nv_bfloat16, true>(p, c.stream))
                                                      : (f16 ? gather_go<__half, false>(p, c.stream) : gather_go<__nv_bfloat16, false>(p, c.stream));
  if (!cuda_ok(e, who)) return c.err;
  count_launch("kv_gather_kernel");
  return PULPNN_OK;
}
