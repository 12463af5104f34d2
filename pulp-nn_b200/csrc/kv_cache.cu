// kv_cache.cu -- rows into and out of a paged cache of keys and values: pulpnn_kv_append (position rotation of
// queries and keys, storing with a cut to 8 bits) and pulpnn_kv_gather.
//
// Both move bytes: 48 rows of 128 channels a token at 32 query and 8 key heads, some 4 operations a channel. A row is
// held by 16 lanes (8 for heads of up to 64 channels), 8 channels each, so that a warp loads and stores whole rows in
// 16-byte pieces and a row's largest value is 4 (3) shuffles away.
#include "attention.cuh"

namespace pulpnn {
namespace attn {

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

constexpr int THREADS = 256;

struct AppendProblem {
  const char *in[3];          // q, k, v
  char *out[3];
  const float *step[3];
  int64_t in_token[3], in_head[3], out_token[3], out_head[3];      // bytes
  const long long *slots;
  const int *positions;
  const double *inv_freq;
  CacheView cache;
  int n, hq, rows, dim, rot, half;
};

struct S32 {};
struct F32 {};
template <typename IN> struct InSize { static constexpr int v = 2; };
template <> struct InSize<S32> { static constexpr int v = 4; };
template <> struct InSize<F32> { static constexpr int v = 4; };

// one channel, and eight from a 16-byte boundary (S32 before the step)
template <typename IN> __device__ __forceinline__ float load1(const char *p) { return (float)*reinterpret_cast<const IN *>(p); }
template <> __device__ __forceinline__ float load1<S32>(const char *p) { return (float)*reinterpret_cast<const int *>(p); }
template <> __device__ __forceinline__ float load1<F32>(const char *p) { return *reinterpret_cast<const float *>(p); }
template <typename IN> __device__ __forceinline__ void load8(const char *p, float (&x)[8])
{
  const uint4 w = *reinterpret_cast<const uint4 *>(p);
  const float2 a = unpack2<IN>(w.x), b = unpack2<IN>(w.y), c = unpack2<IN>(w.z), d = unpack2<IN>(w.w);
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
}
template <> __device__ __forceinline__ void load8<S32>(const char *p, float (&x)[8])
{
  const int4 a = reinterpret_cast<const int4 *>(p)[0], b = reinterpret_cast<const int4 *>(p)[1];
  x[0] = (float)a.x; x[1] = (float)a.y; x[2] = (float)a.z; x[3] = (float)a.w;
  x[4] = (float)b.x; x[5] = (float)b.y; x[6] = (float)b.z; x[7] = (float)b.w;
}
template <> __device__ __forceinline__ void load8<F32>(const char *p, float (&x)[8])
{
  const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
// times the real value of a step, channel by channel
__device__ __forceinline__ void times8(const float *step, float (&x)[8])
{
  float s[8];
  if ((reinterpret_cast<uintptr_t>(step) & 15) == 0) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(step)), b = __ldg(reinterpret_cast<const float4 *>(step) + 1);
    s[0] = a.x; s[1] = a.y; s[2] = a.z; s[3] = a.w; s[4] = b.x; s[5] = b.y; s[6] = b.z; s[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) s[i] = __ldg(step + i);
  }
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] *= s[i];
}

// One block: the rows blockIdx.y, blockIdx.y + gridDim.y, ... (in groups of THREADS / LANES) of one token.
template <typename IN, typename WIDE, bool EIGHT, int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS) kv_append_kernel(const AppendProblem p)
{
  constexpr int SIZE = InSize<IN>::v, PER = THREADS / LANES;
  __shared__ float2 turn[MAX_HEAD_DIM / 2];
  const int token = blockIdx.x, lane = threadIdx.x % LANES, sub = threadIdx.x / LANES, c0 = lane * 8;
  pdl_wait();
  if (threadIdx.x < p.half) {
    // The angle in turns, in 64 bits: a position of 10^5 times a frequency near 1 leaves 32 bits with errors of 10^-2.
    // Its fraction of a turn keeps 24 bits, and sincospif takes multiples of pi.
    const double turns = (double)__ldg(p.positions + token) * __ldg(p.inv_freq + threadIdx.x) * 0.15915494309189533577;
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    turn[threadIdx.x] = make_float2(c, s);
  }
  const long long slot = __ldg(p.slots + token);
  const bool stored = slot >= 0 && slot < p.cache.n_slots;
  const int page = stored ? p.cache.by_page.div((int)slot) : 0, at = stored ? (int)slot - page * p.cache.page_size : 0;
  __syncthreads();
  // the bound is a whole number of warps: all lanes of a row stay together
  for (int row0 = blockIdx.y * PER; row0 < p.rows; row0 += gridDim.y * PER) {
    const int row = row0 + sub;
    const bool live = row < p.rows && c0 < p.dim;
    const int which = row < p.hq ? 0 : (row < p.hq + p.cache.n_heads ? 1 : 2);
    const int head = row - (which == 0 ? 0 : (which == 1 ? p.hq : p.hq + p.cache.n_heads));
    float x[8], y[8];
    if (live) {
      const char *src = p.in[which] + token * p.in_token[which] + head * p.in_head[which] + c0 * SIZE;
      const float *step = sizeof(IN) == 1 && p.step[which] ? p.step[which] + (int64_t)head * p.dim + c0 : nullptr;
      load8<IN>(src, x);
      if (step) times8(step, x);
      if (which < 2 && c0 < p.rot) {
        if (INTERLEAVED) {
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            if (c0 + i < p.rot) {
              const float2 t = turn[(c0 + i) >> 1];
              y[i] = x[i] * t.x - x[i + 1] * t.y;
              y[i + 1] = x[i + 1] * t.x + x[i] * t.y;
            } else { y[i] = x[i]; y[i + 1] = x[i + 1]; }
          }
        } else if ((p.half & 7) == 0) {
          // the other channels of the eight pairs are eight of one other lane, which has loaded them too
          const bool low = c0 < p.half;
          const int other = low ? p.half : -p.half, i0 = low ? c0 : c0 - p.half;
          float z[8];
          load8<IN>(src + other * SIZE, z);
          if (step) times8(step + other, z);
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float2 t = turn[i0 + i];
            y[i] = x[i] * t.x + (low ? -z[i] : z[i]) * t.y;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int c = c0 + i;
            y[i] = x[i];
            if (c < p.rot) {
              const bool low = c < p.half;
              const int other = low ? p.half : -p.half;
              float z = load1<IN>(src + (i + other) * SIZE);
              if (step) z *= __ldg(step + i + other);
              const float2 t = turn[low ? c : c - p.half];
              y[i] = x[i] * t.x + (low ? -z : z) * t.y;
            }
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = x[i];
      }
    }
    __syncwarp();              // in place: every lane of the row has read what another lane now writes over
    const uint4 wide = live ? make_uint4(pack2<WIDE>(y[0], y[1]), pack2<WIDE>(y[2], y[3]), pack2<WIDE>(y[4], y[5]),
                                         pack2<WIDE>(y[6], y[7])) : make_uint4(0, 0, 0, 0);
    if (live && p.out[which])
      *reinterpret_cast<uint4 *>(p.out[which] + token * p.out_token[which] + head * p.out_head[which] + c0 * 2) = wide;
    if (EIGHT) {
      float most = 0.f;
      bool odd = false;
      if (live) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          most = fmaxf(most, fabsf(y[i]));
          odd |= !(fabsf(y[i]) <= 3.402823466e38f);
        }
      }
      if (odd) most = __int_as_float(0x7f800000);
#pragma unroll
      for (int d = 1; d < LANES; d *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
      if (live && which > 0 && stored) {
        const bool fine = most <= 3.402823466e38f, any = most >= 7.888609e-31f && fine;     // 2^-100
        const float inv = any ? 127.f / most : 0.f;
        int q[8];
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = any ? min(max(__float2int_rn(y[i] * inv), -127), 127) : 0;
        uint2 w;
        w.x = (q[0] & 255) | (q[1] & 255) << 8 | (q[2] & 255) << 16 | (unsigned)q[3] << 24;
        w.y = (q[4] & 255) | (q[5] & 255) << 8 | (q[6] & 255) << 16 | (unsigned)q[7] << 24;
        char *base = which == 1 ? p.cache.k : p.cache.v;
        *reinterpret_cast<uint2 *>(base + row_of(p.cache, page, at, head) + c0) = w;
        if (lane == 0)
          (which == 1 ? p.cache.k_scale : p.cache.v_scale)[scale_of(p.cache, page, at, head)] =
              any ? most / 127.f : (fine ? 0.f : __int_as_float(0x7fffffff));
      }
    } else if (live && which > 0 && stored) {
      char *base = which == 1 ? p.cache.k : p.cache.v;
      *reinterpret_cast<uint4 *>(base + (row_of(p.cache, page, at, head) + c0) * 2) = wide;
    }
  }
}

template <typename IN, typename WIDE, bool EIGHT>
cudaError_t append_go(const AppendProblem &p, bool interleaved, dim3 grid, cudaStream_t s)
{
  const bool narrow = p.dim <= 64;
  auto k = narrow ? (interleaved ? kv_append_kernel<IN, WIDE, EIGHT, 8, true> : kv_append_kernel<IN, WIDE, EIGHT, 8, false>)
                  : (interleaved ? kv_append_kernel<IN, WIDE, EIGHT, 16, true> : kv_append_kernel<IN, WIDE, EIGHT, 16, false>);
  return launch_pdl(k, grid, dim3(THREADS), 0, s, p);
}
template <typename WIDE, bool EIGHT>
cudaError_t append_in(int in_type, const AppendProblem &p, bool interleaved, dim3 grid, cudaStream_t s)
{
  switch (in_type) {
    case PULPNN_TYPE_F16: return append_go<__half, WIDE, EIGHT>(p, interleaved, grid, s);
    case PULPNN_TYPE_BF16: return append_go<__nv_bfloat16, WIDE, EIGHT>(p, interleaved, grid, s);
    case PULPNN_TYPE_F32: return append_go<F32, WIDE, EIGHT>(p, interleaved, grid, s);
    default: return append_go<S32, WIDE, EIGHT>(p, interleaved, grid, s);
  }
}

struct GatherProblem {
  const long long *slots;
  char *out[2];
  int64_t out_token[2], out_head[2];      // bytes
  CacheView cache;
  int n, dim;
};

// One row of 8 channels a lane; blockIdx.y is the head, blockIdx.z keys or values.
template <typename WIDE, bool EIGHT, int LANES>
__global__ void __launch_bounds__(THREADS) kv_gather_kernel(const GatherProblem p)
{
  constexpr int PER = THREADS / LANES;
  const int lane = threadIdx.x % LANES, c0 = lane * 8, head = blockIdx.y, which = p.out[0] ? blockIdx.z : 1;
  const int64_t token = (int64_t)blockIdx.x * PER + threadIdx.x / LANES;
  pdl_wait();
  if (token >= p.n || c0 >= p.dim) return;
  const long long slot = __ldg(p.slots + token);
  uint4 w = make_uint4(0, 0, 0, 0);
  if (slot >= 0 && slot < p.cache.n_slots) {
    const int page = p.cache.by_page.div((int)slot), at = (int)slot - page * p.cache.page_size;
    const char *base = which == 0 ? p.cache.k : p.cache.v;
    if (EIGHT) {
      const uint2 q = *reinterpret_cast<const uint2 *>(base + row_of(p.cache, page, at, head) + c0);
      const float s = (which == 0 ? p.cache.k_scale : p.cache.v_scale)[scale_of(p.cache, page, at, head)];
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = (float)(signed char)((i < 4 ? q.x : q.y) >> (8 * (i & 3))) * s;
      w = make_uint4(pack2<WIDE>(x[0], x[1]), pack2<WIDE>(x[2], x[3]), pack2<WIDE>(x[4], x[5]), pack2<WIDE>(x[6], x[7]));
    } else {
      w = *reinterpret_cast<const uint4 *>(base + (row_of(p.cache, page, at, head) + c0) * 2);
    }
  }
  *reinterpret_cast<uint4 *>(p.out[which] + token * p.out_token[which] + head * p.out_head[which] + c0 * 2) = w;
}

template <typename WIDE, bool EIGHT>
cudaError_t gather_go(const GatherProblem &p, cudaStream_t s)
{
  const int lanes = p.dim <= 64 ? 8 : 16, per = THREADS / lanes;
  const dim3 grid((unsigned)((p.n + per - 1) / per), (unsigned)p.cache.n_heads, p.out[0] && p.out[1] ? 2 : 1);
  return lanes == 8 ? launch_pdl(kv_gather_kernel<WIDE, EIGHT, 8>, grid, dim3(THREADS), 0, s, p)
                    : launch_pdl(kv_gather_kernel<WIDE, EIGHT, 16>, grid, dim3(THREADS), 0, s, p);
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
  ATTN_REQUIRE(cache->type == PULPNN_TYPE_S8 || cache->type == a->out_type, PULPNN_ERR_UNSUPPORTED,
               "%s: a 16-bit cache of another type than out_type", who);
  ATTN_REQUIRE((a->q != nullptr) == (a->q_out != nullptr), PULPNN_ERR_INVALID_ARG, "%s: q without q_out, or q_out without q", who);
  ATTN_REQUIRE(!a->q || (a->n_q_heads > 0 && a->n_q_heads <= 65535), PULPNN_ERR_INVALID_ARG, "%s: %d query heads", who, a->n_q_heads);
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
    p.in[i] = static_cast<const char *>(in[i]); p.out[i] = static_cast<char *>(out[i]); p.step[i] = s32 ? step[i] : nullptr;
    p.in_token[i] = is_[i][0] * is; p.in_head[i] = is_[i][1] * is;
    p.out_token[i] = os[i][0] * 2; p.out_head[i] = os[i][1] * 2;
  }
  p.slots = reinterpret_cast<const long long *>(a->slots); p.positions = a->positions; p.inv_freq = a->inv_freq;
  p.cache = view_of(*cache);
  p.n = a->n_tokens; p.hq = a->q ? a->n_q_heads : 0; p.rows = p.hq + 2 * cache->n_heads; p.dim = cache->head_dim;
  p.rot = a->rotary_dim; p.half = a->rotary_dim / 2;
  // Few tokens: a block for every group of rows, so that a single token's rows are in flight together. Many: one block
  // a token, which computes the token's angles once.
  const int per = THREADS / (p.dim <= 64 ? 8 : 16), groups = (p.rows + per - 1) / per;
  const dim3 grid((unsigned)p.n, (unsigned)(p.n < 4 * c.sm_count ? groups : 1));
  const bool il = a->interleaved != 0, f16 = a->out_type == PULPNN_TYPE_F16;
  const cudaError_t e = cache->type == PULPNN_TYPE_S8
      ? (f16 ? append_in<__half, true>(a->in_type, p, il, grid, c.stream) : append_in<__nv_bfloat16, true>(a->in_type, p, il, grid, c.stream))
      : (f16 ? append_in<__half, false>(a->in_type, p, il, grid, c.stream) : append_in<__nv_bfloat16, false>(a->in_type, p, il, grid, c.stream));
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
