// attn_decode.cu -- pulpnn_attn_decode: one new token per sequence against a paged cache of keys and values.
//
//   o[b][h] = sum_t w_t v[t],  w = softmax over t of scale * (q[b][h] . k[t]),  t the last `window` tokens of sequence b.
//
// Every key and value is read once and used for the G query heads that share it: 4 G operations on 2 or 4 bytes, so the
// kernel is bound by memory as long as the arithmetic stays out of the way. That is on the tensor cores
// (mma.m16n8k16): S^T = K Q^T with 16 tokens as the rows and 8 query heads as the columns, and O^T = V^T P^T with 16
// channels as the rows. With the heads as columns a group of up to 8 wastes half as much as it would as rows, and the
// weights only have to be transposed in 8x8 blocks (movmatrix) on their way from the one product to the other. tcgen05
// would want 128 rows, M = tokens, for 16 bytes of results each: it reads its operands from shared memory just the
// same, and its accumulators would have to come back through TMEM for the running maximum.
//
// A warp works alone: tiles of 16 (8-bit or up to 64 channels: 32) tokens, fetched by itself into STAGES buffers of its own;
// there is no barrier between warps until the end. Each lane looks up the page of one token, one tile ahead of its
// fetch. Where pages are a multiple of 16 slots, every 16 tokens lie in one page and come by one TMA copy for each 128 bytes of
// their rows: copies of 16 bytes with a page each cost as many instructions as all the arithmetic. Pages of any
// other size are fetched with these (16-byte cp.async), tokens behind the end without being read.
//
// WARPS warps are a CTA, up to eight CTAs of a cluster share a sequence, and the partial results are joined through
// (distributed) shared memory. Where clusters of eight are too few to fill the GPU, several share a sequence and leave
// their sums in memory for attn_join_kernel: memory from a pool, allocated and freed in the stream's order, so that calls
// on other streams and replays of other graphs have their own. Every join goes in a fixed order, without atomics: the
// same result every time.
//
// Measured (one B200; the copy rate is 6.56 TB/s): 64 ragged sequences of up to 8192 tokens, 32 query and 8 key heads of 128
// channels in 16 bits, 166 us (6.6 TB/s); 8 of 128k in 8 bits 330 us (6.5 TB/s; 178 M instructions, issue slots 56 % busy),
// 375 in a long run, where the power limit lowers the clock; 200 with a window of 1024, 16 heads of 80 channels, pages of 20
// slots, 136 us (6.1 TB/s: 64 tiles a sequence, so that the CTAs' starts and joins show); one of 131072 tokens and 8 heads
// 90 us (6.0 TB/s); one of 1000 tokens 6.3 us, a chain of six round trips to memory and two cluster barriers.
//
// Running maximum: the reference m only has to be near the true maximum, not equal to it. It is raised (and the sums
// rescaled) when some weight would be above 2^LAG, which one vote per tile finds out; the weights stay
// below that, which the 16-bit types hold, and the sums are kept in 32 bits. fp16 ends at 2^-24 on the other side, and many small
// weights make a sum: there the reference is set 2^UNDER below the maximum, so that weights down to 2^-21 of the largest one keep
// all their bits, and each is off by 2^-32 of it at most. It is raised as often as with 8 and 0, bf16's.
//
// 8-bit caches: codes are exact in fp16, so K's product is exact but for q, whose rows are scaled by a power of two
// to a maximum of 1 .. 2 (bf16 queries lose nothing that matters: 2^-24 of the row's maximum). The key's scale
// multiplies the score. The value's scale multiplies the weight before it is rounded to fp16; such weights get a reference of
// their own, the running maximum of score + log2(scale), so that they keep fp16's 11 bits whatever the scales are.
#include <cooperative_groups.h>

#include "attention.cuh"
#include "sm100_primitives.cuh"

namespace pulpnn {
namespace attn {
namespace {

namespace cg = cooperative_groups;

// Two stages of 8 KB a warp and three CTAs an SM: twelve warps keep 96 KB under way and two thirds of the issue slots busy where
// the cache holds 8 bits. Three stages and two CTAs: 171 instead of 165 us for 64 ragged sequences of up to 8192 tokens in
// 16 bits, 189 instead of 151 for 200 of 80 channels.
constexpr int WARPS = 4, STAGES = 2, MOST_SPLITS = 8;
constexpr float NOTHING = -3.402823466e38f;       // the lowest number: any score is at least that
template <typename T> struct Room { static constexpr float LAG = 15.f, UNDER = 7.f; };
template <> struct Room<__nv_bfloat16> { static constexpr float LAG = 8.f, UNDER = 0.f; };

struct DecodeProblem {
  const char *q;
  char *out;
  float *lse;
  const int *table, *lens;
  int64_t q_seq, q_head, out_seq, out_head;      // bytes
  int64_t table_stride;
  CacheView cache;
  int hq, group, head_tiles, dim, max_pages, window, q_type, out_type;
  float scale_log2, out_inv_step;
  int out_zero, splits, parts;                   // CTAs of a cluster, clusters of a sequence
  float *sums;                                   // parts > 1: [pair][part][Partial]
  int box;                                       // tokens of a TMA copy: 16 or a whole tile
  int *status;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool live)
{
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, bool live)
{
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix4(uint32_t a, unsigned (&r)[4])
{
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t a, unsigned (&r)[4])
{
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// two 16x16 blocks of bytes, transposed: a lane's word i of a block holds column g + 8 i of rows 4t .. 4t + 3
__device__ __forceinline__ void ldmatrix2_trans8(uint32_t a, unsigned (&r)[4])
{
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ unsigned transpose8(unsigned a)
{
  unsigned d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ unsigned lds32(uint32_t a)
{
  unsigned v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float ex2(float x)
{
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T> __device__ __forceinline__ void mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1);
template <> __device__ __forceinline__ void mma<__half>(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1)
{
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1)
{
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float load_q(const char *p, int type)
{
  return type == PULPNN_TYPE_F16 ? __half2float(*reinterpret_cast<const __half *>(p)) : __bfloat162float(*reinterpret_cast<const __nv_bfloat16 *>(p));
}

// Rows of 128 bytes (a box of 64 16-bit channels or of up to 128 8-bit ones), whose 16-byte chunks are swizzled by their row the way
// TMA does it: eight rows of one chunk lie in different banks. DENSE: rows as long as they are, two of eight in the same banks,
// where a second box of 64 channels would be mostly empty: 41 KB a CTA instead of 66, five of them an SM instead of three
// (the 200 sequences above: 139 us, 153 in two boxes).
template <int DP, bool EIGHT> struct Tile {
  static constexpr int SIZE = EIGHT ? 1 : 2;
  static constexpr int TOKENS = EIGHT || DP <= 64 ? 32 : 16;
  static constexpr bool DENSE = !EIGHT && DP == 80;
  static constexpr int BOXES = EIGHT || DP <= 64 || DENSE ? 1 : 2;
  static constexpr int BOX = TOKENS * (DENSE ? DP * 2 : 128);    // bytes
  static constexpr int CHUNKS = DP * SIZE / 16;              // of a row
  static constexpr int STAGE = 2 * BOXES * BOX;              // keys, values
  static constexpr int PIPE = WARPS * STAGES * STAGE;
  static constexpr int SCALES = EIGHT ? WARPS * STAGES * 2 * TOKENS * 4 : 0;
  // address of a 16-byte chunk of a token's row, from the tile's first byte
  static __device__ __forceinline__ uint32_t at(int token, int chunk)
  {
    if (DENSE) return token * (DP * 2) + chunk * 16;
    return (BOXES > 1 ? (chunk >> 3) * BOX : 0) + token * 128 + (((chunk & 7) ^ (token & 7)) << 4);
  }
};
// what the join needs, in the pipeline's place: per warp [heads][DP] sums, then the CTA's
template <int DP, int NT> struct Join {
  static constexpr int HEADS = NT * 8, PITCH = DP + 4;
  static constexpr int WARP = HEADS * PITCH;                 // floats
  static constexpr int STATS = 3 * HEADS;                    // m, l, reference of the sums
  static constexpr int BYTES = (WARPS * (WARP + STATS) + WARP + STATS) * 4;
};
// dynamic shared memory: the pipeline, or the join in its place; the scales; room to align the whole
template <int DP, int NT, bool EIGHT> struct Smem {
  static constexpr int PIPE = Tile<DP, EIGHT>::PIPE > Join<DP, NT>::BYTES ? Tile<DP, EIGHT>::PIPE : Join<DP, NT>::BYTES;
  static constexpr int BYTES = PIPE + Tile<DP, EIGHT>::SCALES + 1024;
};

// what a cluster leaves behind: sums [8 NT heads][MAX_HEAD_DIM], and m, l and the sums' reference of each head
__host__ __device__ constexpr int partial_floats(int nt) { return nt * 8 * (MAX_HEAD_DIM + 4); }

// A block for each head and sequence: joins the parts, a channel a thread.
template <int NT>
__global__ void __launch_bounds__(MAX_HEAD_DIM) attn_join_kernel(const DecodeProblem p)
{
  pdl_wait();
  const int pair = blockIdx.x, head = blockIdx.y, ch = threadIdx.x;
  const int ht = pair % p.head_tiles, kvh = pair / p.head_tiles % p.cache.n_heads, seq = pair / p.head_tiles / p.cache.n_heads;
  if (head >= min(NT * 8, p.group - ht * NT * 8)) return;
  const float *sums = p.sums + (int64_t)pair * p.parts * partial_floats(NT);
  float M = NOTHING, R = NOTHING, L = 0.f, acc = 0.f;
  for (int i = 0; i < p.parts; i++) {
    const float *st = sums + i * partial_floats(NT) + NT * 8 * MAX_HEAD_DIM;
    M = fmaxf(M, st[head]);
    R = fmaxf(R, st[2 * NT * 8 + head]);
  }
  for (int i = 0; i < p.parts; i++) {
    const float *st = sums + i * partial_floats(NT) + NT * 8 * MAX_HEAD_DIM;
    L += st[NT * 8 + head] * ex2(st[head] - M);
    if (ch < p.dim) acc += sums[i * partial_floats(NT) + head * MAX_HEAD_DIM + ch] * ex2(st[2 * NT * 8 + head] - R);
  }
  const float y = L == 0.f ? 0.f : acc * (ex2(R - M) / L);
  const int h = kvh * p.group + ht * NT * 8 + head;
  char *dst = p.out + seq * p.out_seq + (int64_t)h * p.out_head;
  if (ch < p.dim) {
    if (p.out_type == PULPNN_TYPE_U8) dst[ch] = (char)to_u8(y, p.out_inv_step, p.out_zero);
    else if (p.out_type == PULPNN_TYPE_F16) reinterpret_cast<__half *>(dst)[ch] = __float2half_rn(y);
    else reinterpret_cast<__nv_bfloat16 *>(dst)[ch] = __float2bfloat16_rn(y);
  }
  if (p.lse && ch == 0) p.lse[(int64_t)seq * p.hq + h] = (M + log2f(L)) * 0.69314718055994530942f;
}

template <typename T, int DP, int NT, bool EIGHT, bool TMA>
__global__ void __launch_bounds__(WARPS * 32)
attn_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const DecodeProblem p)
{
  using TL = Tile<DP, EIGHT>;
  using JN = Join<DP, NT>;
  constexpr int KS = DP / 16, MT = TL::TOKENS / 16;
  constexpr float LAG = Room<T>::LAG, UNDER = Room<T>::UNDER;
  extern __shared__ char raw[];
  __shared__ uint64_t full[WARPS][STAGES];
  __shared__ int abort_flag;
  char *smem = raw + (((sm100::smem_u32(raw) + 1023u) & ~1023u) - sm100::smem_u32(raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = blockIdx.x % p.splits;
  int rest = blockIdx.x / p.splits;
  const int cluster_id = rest, part = rest % p.parts;
  rest /= p.parts;
  const int ht = rest % p.head_tiles; rest /= p.head_tiles;
  const int kvh = rest % p.cache.n_heads, seq = rest / p.cache.n_heads;
  const int h0 = kvh * p.group + ht * NT * 8, heads = min(NT * 8, p.group - ht * NT * 8);

  if (TMA) {
    if (threadIdx.x == 0) {
      abort_flag = 0;
      for (int i = 0; i < WARPS * STAGES; i++) sm100::mbar_init(&full[0][0] + i, 1);
      sm100::mbar_fence_init();
    }
    __syncthreads();
  } else if (p.dim < DP) {       // channels behind the head's own stay zero: a NaN there would spoil the product with q's zeros
    for (int i = threadIdx.x; i < TL::PIPE / 16; i += WARPS * 32) reinterpret_cast<uint4 *>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  pdl_wait();
  const int n = min(max(__ldg(p.lens + seq), 0), p.max_pages * p.cache.page_size);
  const int first = p.window > 0 ? max(0, n - p.window) : 0, origin = TMA ? first & ~15 : first;      // of the tiles
  const int tiles = (n - origin + TL::TOKENS - 1) / TL::TOKENS;
  const int share = part * p.splits + rank, shares = p.parts * p.splits;
  const int lo = (int)((int64_t)tiles * share / shares), hi = (int)((int64_t)tiles * (share + 1) / shares);
  const int mine = hi - lo > warp ? (hi - lo - warp + WARPS - 1) / WARPS : 0;       // tiles lo + warp + i * WARPS

  char *pipe_at = smem + warp * STAGES * TL::STAGE;
  const uint32_t pipe = sm100::smem_u32(pipe_at);
  const uint32_t scales = sm100::smem_u32(smem) + Smem<DP, NT, EIGHT>::PIPE + warp * STAGES * 2 * TL::TOKENS * 4;
  const int *table = p.table + seq * p.table_stride;
  // the page of this lane's token of tile i; -1 where there is none
  auto page_of = [&](int i, int &at) -> int {
    const int token = origin + (lo + warp + i * WARPS) * TL::TOKENS + (lane & (TL::TOKENS - 1));
    at = 0;
    if (i >= mine || token >= n) return -1;
    const int in_row = p.cache.by_page.div(token), page = __ldg(table + in_row);
    at = token - in_row * p.cache.page_size;
    return page >= 0 && page < p.cache.n_pages ? page : -1;
  };
  unsigned live_ring = 0;      // bit `stage`: whether this lane's token of that stage counts
  auto fetch = [&](int i, int page, int at) {
    const int stage = i % STAGES;
    const uint32_t base = pipe + stage * TL::STAGE;
    const bool live = page >= 0 && (!TMA || origin + (lo + warp + i * WARPS) * TL::TOKENS + (lane & (TL::TOKENS - 1)) >= first);
    live_ring = (live_ring & ~(1u << stage)) | (live ? 1u << stage : 0u);
    if (i < mine) {
      if (TMA) {
        // a page that is none lies outside the map, and its rows become zero
        const int page16 = TL::TOKENS > 16 ? __shfl_sync(0xffffffffu, page, 16) : 0, at16 = TL::TOKENS > 16 ? __shfl_sync(0xffffffffu, at, 16) : 0;
        if (lane == 0) {
          uint64_t *bar = &full[warp][stage];
          char *dst = pipe_at + stage * TL::STAGE;
          sm100::mbar_arrive_expect_tx(bar, TL::STAGE);
#pragma unroll
          for (int b = 0; b < TL::BOXES; b++) {
            sm100::tma_load_4d(dst + b * TL::BOX, &map_k, bar, b * 64, at, kvh, page);
            sm100::tma_load_4d(dst + (TL::BOXES + b) * TL::BOX, &map_v, bar, b * 64, at, kvh, page);
            if (TL::TOKENS > 16 && p.box == 16) {
              sm100::tma_load_4d(dst + b * TL::BOX + 2048, &map_k, bar, b * 64, at16, kvh, page16);
              sm100::tma_load_4d(dst + (TL::BOXES + b) * TL::BOX + 2048, &map_v, bar, b * 64, at16, kvh, page16);
            }
          }
        }
      } else {
        const int64_t off = live ? row_of(p.cache, page, at, kvh) * TL::SIZE : 0;
#pragma unroll
        for (int j = 0; j < TL::TOKENS * TL::CHUNKS / 32; j++) {
          const int item = lane + 32 * j, row = item / TL::CHUNKS, chunk = item % TL::CHUNKS;
          const int64_t o = __shfl_sync(0xffffffffu, off, row);
          const bool ok = __shfl_sync(0xffffffffu, live, row);
          if (chunk * 16 < p.dim * TL::SIZE) {
            cp_async16(base + TL::at(row, chunk), p.cache.k + (ok ? o + chunk * 16 : 0), ok);
            cp_async16(base + TL::BOXES * TL::BOX + TL::at(row, chunk), p.cache.v + (ok ? o + chunk * 16 : 0), ok);
          }
        }
      }
      if (EIGHT) {
        const int64_t s = live ? scale_of(p.cache, page, at, kvh) : 0;
        cp_async4(scales + (stage * 2 * TL::TOKENS + lane) * 4, p.cache.k_scale + s, live);
        cp_async4(scales + ((stage * 2 + 1) * TL::TOKENS + lane) * 4, p.cache.v_scale + s, live);
      }
    }
    if (EIGHT || !TMA) cp_commit();
  };
  int page_next, at_next;
  {
    int page[STAGES], at[STAGES];
#pragma unroll
    for (int i = 0; i < STAGES; i++) page[i] = page_of(i, at[i]);
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) fetch(i, page[i], at[i]);
    page_next = page[STAGES - 1]; at_next = at[STAGES - 1];
  }

  // q as the second operand: head g of each tile of 8, channels 16 ks + {2t, 2t+1} and {2t+8, 2t+9}; 8-bit: 4t .. 4t+3
  unsigned qf[NT][KS][2];
  float q_scale[NT][2];        // of this thread's heads 2t, 2t+1 in the accumulators
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const bool live = nt * 8 + g < heads;
    const char *row = p.q + seq * p.q_seq + (int64_t)(h0 + nt * 8 + g) * p.q_head;
    if (!EIGHT) {
#pragma unroll
      for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int half = 0; half < 2; half++) {
          const int c = ks * 16 + half * 8 + 2 * t;
          qf[nt][ks][half] = live && c < p.dim ? *reinterpret_cast<const unsigned *>(row + c * 2) : 0u;
        }
      q_scale[nt][0] = q_scale[nt][1] = p.scale_log2;
    } else {
      float x[KS][4], most = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int c = ks * 16 + 4 * t + e;
          x[ks][e] = live && c < p.dim ? load_q(row + c * 2, p.q_type) : 0.f;
          most = fmaxf(most, fabsf(x[ks][e]));
        }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // the power of two at or below the row's maximum (1 for a row of zeros, infinities or the smallest numbers); one over it is
      // 2^-127 for the largest, a number below the normal ones
      const unsigned e = (__float_as_uint(most) >> 23) & 255u;
      const bool fits = e >= 1 && e <= 254;
      const float up = fits ? __uint_as_float(e < 254 ? (254u - e) << 23 : 1u << 22) : 1.f, down = fits ? __uint_as_float(e << 23) : 1.f;
#pragma unroll
      for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int half = 0; half < 2; half++) qf[nt][ks][half] = pack2<__half>(x[ks][2 * half] * up, x[ks][2 * half + 1] * up);
#pragma unroll
      for (int c = 0; c < 2; c++) q_scale[nt][c] = __shfl_sync(0xffffffffu, down, (2 * t + c) * 4) * p.scale_log2;
    }
  }

  float o[NT][KS][4], m[NT][2], l[NT][2], ref[NT][2];       // ref: the reference of the sums o; m's own where a cache is 16 bits wide
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int e = 0; e < 4; e++) o[nt][ks][e] = 0.f;
    m[nt][0] = m[nt][1] = ref[nt][0] = ref[nt][1] = NOTHING;
    l[nt][0] = l[nt][1] = 0.f;
  }

  // Which of 16 tokens are rows g and g + 8 of the products' fragments. 8-bit: the transposed load gives a lane tokens 4t .. 4t + 3,
  // of which two follow from rows 2t and 2t + 1 of the first eight and two from the second eight; t >= 2 has them the other
  // way round, so that the first eight rows of a key load lie in different banks.
  auto token_of = [&](int r) { return EIGHT ? 4 * (g >> 1) + ((g >> 2) ^ r) * 2 + (g & 1) : r * 8 + g; };
  const int k_row = 4 * ((lane & 7) >> 1) + ((((lane & 7) >> 2) ^ ((lane >> 3) & 1)) * 2) + (lane & 1);
  const unsigned first_two = t < 2 ? 0x4140 : 0x4342, last_two = t < 2 ? 0x4342 : 0x4140;
  bool landed = true;
  for (int i = 0; i < mine; i++) {
    const int stage = i % STAGES;
    fetch(i + STAGES - 1, page_next, at_next);
    page_next = page_of(i + STAGES, at_next);
    if (EIGHT || !TMA) cp_wait<STAGES - 1>();
    if (TMA) landed = sm100::mbar_wait(&full[warp][stage], (i / STAGES) & 1, &abort_flag, p.status, 1 << 25) && landed;
    __syncwarp();
    const uint32_t base = pipe + stage * TL::STAGE, vbase = base + TL::BOXES * TL::BOX, sbase = scales + stage * 2 * TL::TOKENS * 4;
    const unsigned live = __ballot_sync(0xffffffffu, (live_ring >> stage) & 1u);
    if (TMA && !EIGHT && live != 0xffffffffu) {
      // a page's rows that are not this sequence's tokens: a weight of 0 does not keep an infinity or a NaN out of the sum
      if (!((live >> lane) & 1u) && lane < TL::TOKENS) {
#pragma unroll
        for (int c = 0; c < TL::CHUNKS; c++) sm100::sts128(vbase + TL::at(lane, c), 0, 0, 0, 0);
      }
      sm100::fence_proxy_async();
      __syncwarp();
    }

    // S^T: tokens 16 mt + {token_of(0), token_of(1)} x heads 8 nt + {2t, 2t + 1}
    float s[MT][NT][4];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[mt][nt][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ks += EIGHT ? 2 : 1) {
        unsigned a[4];
        if (EIGHT) {
          unsigned w[4];
          ldmatrix4(base + TL::at(mt * 16 + k_row, ks + (lane >> 4)), w);
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const unsigned w0 = w[2 * e] ^ 0x80808080u, w1 = w[2 * e + 1] ^ 0x80808080u;
            a[0] = widen(w0, 0x4140); a[1] = widen(w1, 0x4140); a[2] = widen(w0, 0x4342); a[3] = widen(w1, 0x4342);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) mma<T>(s[mt][nt], a, qf[nt][ks + e][0], qf[nt][ks + e][1]);
          }
        } else {
          ldmatrix4(base + TL::at(mt * 16 + (lane & 15), ks * 2 + (lane >> 4)), a);
#pragma unroll
          for (int nt = 0; nt < NT; nt++) mma<T>(s[mt][nt], a, qf[nt][ks][0], qf[nt][ks][1]);
        }
      }
    }
    float vs[MT][2], lvs[MT][2];
    bool over = false;
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const int token = mt * 16 + token_of(r);
        const bool ok = (live >> token) & 1u;
        float ks_ = 1.f;
        if (EIGHT) {
          ks_ = __uint_as_float(lds32(sbase + token * 4));
          vs[mt][r] = __uint_as_float(lds32(sbase + (TL::TOKENS + token) * 4));
          lvs[mt][r] = __log2f(fabsf(vs[mt][r]));
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int c = 0; c < 2; c++) {
            float &x = s[mt][nt][2 * r + c];
            // the key's scale first: codes of zero give a zero, whatever the two scales are together
            x = ok ? (EIGHT ? x * ks_ : x) * q_scale[nt][c] : -INFINITY;
            over |= x > m[nt][c] + LAG;
            if (EIGHT) over |= x + lvs[mt][r] > ref[nt][c] + LAG;
          }
      }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
          float a = -INFINITY, b = -INFINITY;
#pragma unroll
          for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
              a = fmaxf(a, s[mt][nt][2 * r + c]);
              if (EIGHT) b = fmaxf(b, s[mt][nt][2 * r + c] + lvs[mt][r]);
            }
#pragma unroll
          for (int d = 4; d < 32; d *= 2) {
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, d));
            if (EIGHT) b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, d));
          }
          // the sum of the weights is 32 bits wide wherever its reference lies; an 8-bit cache's has one of its own
          a = fmaxf(m[nt][c], EIGHT ? a : a - UNDER);
          b = EIGHT ? fmaxf(ref[nt][c], b - UNDER) : a;
          l[nt][c] *= ex2(m[nt][c] - a);
          const float f = ex2(ref[nt][c] - b);
          m[nt][c] = a; ref[nt][c] = b;
          // column 2t + c of the accumulators is this thread's in every row
#pragma unroll
          for (int ks = 0; ks < KS; ks++) { o[nt][ks][c] *= f; o[nt][ks][2 + c] *= f; }
        }
    }
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
      unsigned b[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
          float w[2];
#pragma unroll
          for (int c = 0; c < 2; c++) {
            const float x = s[mt][nt][2 * r + c], e = ex2(x - m[nt][c]);
            l[nt][c] += e;
            // rounded to 16 bits for the product with V: off by 2^-8 (bf16) or 2^-11 (fp16) at most; the sum l takes it unrounded
            w[c] = EIGHT ? __uint_as_float(__float_as_uint(ex2(x + lvs[mt][r] - ref[nt][c])) ^ (__float_as_uint(vs[mt][r]) & 0x80000000u)) : e;
          }
          b[nt][r] = transpose8(pack2<T>(w[0], w[1]));
        }
      // O^T += V^T P^T
      if (EIGHT) {
#pragma unroll
        for (int blk = 0; blk < DP / 32; blk++) {
          unsigned w[4];
          ldmatrix2_trans8(vbase + TL::at(mt * 16 + (lane & 15), blk * 2 + (lane >> 4)), w);
#pragma unroll
          for (int e = 0; e < 4; e++) w[e] ^= 0x80808080u;
          const unsigned a0[4] = {widen(w[0], first_two), widen(w[1], first_two), widen(w[0], last_two), widen(w[1], last_two)};
          const unsigned a1[4] = {widen(w[2], first_two), widen(w[3], first_two), widen(w[2], last_two), widen(w[3], last_two)};
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            mma<T>(o[nt][2 * blk], a0, b[nt][0], b[nt][1]);
            mma<T>(o[nt][2 * blk + 1], a1, b[nt][0], b[nt][1]);
          }
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
          unsigned a[4];
          // matrices: (tokens 0-7, channels 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15), each transposed
          ldmatrix4_trans(vbase + TL::at(mt * 16 + (lane & 7) + (lane >> 4) * 8, ks * 2 + ((lane >> 3) & 1)), a);
#pragma unroll
          for (int nt = 0; nt < NT; nt++) mma<T>(o[nt][ks], a, b[nt][0], b[nt][1]);
        }
      }
    }
    __syncwarp();          // the buffer is free for the fetch of the next turn
  }
  cp_wait<0>();
  if (TMA && !landed) {      // given up: what is in flight must land before its memory is used for something else
    volatile int never = 0;
    for (int i = max(0, mine - STAGES); i < mine; i++) sm100::mbar_wait(&full[warp][i % STAGES], (i / STAGES) & 1, &never, nullptr, 0);
  }

  // ---- join: warps, then CTAs of the cluster -----------------------------------------------------
  __syncthreads();         // the pipeline's memory is free
  float *sums = reinterpret_cast<float *>(smem), *stats = sums + WARPS * JN::WARP;
  float *cta_sums = stats + WARPS * JN::STATS, *cta_stats = cta_sums + JN::WARP;
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
#pragma unroll
    for (int c = 0; c < 2; c++) {
      float x = l[nt][c];
#pragma unroll
      for (int d = 4; d < 32; d *= 2) x += __shfl_xor_sync(0xffffffffu, x, d);
      const int head = nt * 8 + 2 * t + c;
      float *st = stats + warp * JN::STATS;
      if (g == 0) { st[head] = m[nt][c]; st[JN::HEADS + head] = x; st[2 * JN::HEADS + head] = ref[nt][c]; }
      float *dst = sums + warp * JN::WARP + head * JN::PITCH;
#pragma unroll
      for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
          const int ch = ks * 16 + r * 8 + g;
          dst[ch] = o[nt][ks][2 * r + c];
        }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < JN::HEADS * DP / 4; i += WARPS * 32) {
    const int head = i / (DP / 4), ch = i % (DP / 4) * 4;
    if (head >= heads) continue;
    float M = NOTHING, R = NOTHING, L = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      M = fmaxf(M, stats[w * JN::STATS + head]);
      R = fmaxf(R, stats[w * JN::STATS + 2 * JN::HEADS + head]);
    }
    float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      const float *st = stats + w * JN::STATS;
      L += st[JN::HEADS + head] * ex2(st[head] - M);
      const float f = ex2(st[2 * JN::HEADS + head] - R);
      const float4 x = *reinterpret_cast<const float4 *>(sums + w * JN::WARP + head * JN::PITCH + ch);
      acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
    }
    *reinterpret_cast<float4 *>(cta_sums + head * JN::PITCH + ch) = acc;
    if (ch == 0) { cta_stats[head] = M; cta_stats[JN::HEADS + head] = L; cta_stats[2 * JN::HEADS + head] = R; }
  }
  // a cluster's barrier, for a CTA alone, is 2 to 5 % of a call with many short sequences
  if (p.splits > 1) cluster.sync();
  else __syncthreads();
  // each CTA writes its share of the outputs, from every CTA's sums
  for (int i = threadIdx.x + rank * WARPS * 32; i < heads * (p.dim / 4); i += p.splits * WARPS * 32) {
    const int head = i / (p.dim / 4), ch = i % (p.dim / 4) * 4;
    float M = NOTHING, R = NOTHING, L = 0.f;
    for (int r = 0; r < p.splits; r++) {
      const float *st = cluster.map_shared_rank(cta_stats, r);
      M = fmaxf(M, st[head]);
      R = fmaxf(R, st[2 * JN::HEADS + head]);
    }
    float4 acc = make_float4(0, 0, 0, 0);
    for (int r = 0; r < p.splits; r++) {
      const float *st = cluster.map_shared_rank(cta_stats, r);
      L += st[JN::HEADS + head] * ex2(st[head] - M);
      const float f = ex2(st[2 * JN::HEADS + head] - R);
      const float4 x = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(cta_sums, r) + head * JN::PITCH + ch);
      acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
    }
    if (p.parts > 1) {
      float *dst = p.sums + (int64_t)cluster_id * partial_floats(NT);
      *reinterpret_cast<float4 *>(dst + head * MAX_HEAD_DIM + ch) = acc;
      dst += NT * 8 * MAX_HEAD_DIM;
      if (ch == 0) { dst[head] = M; dst[NT * 8 + head] = L; dst[2 * NT * 8 + head] = R; }
      continue;
    }
    const float f = L == 0.f ? 0.f : (EIGHT ? ex2(R - M) : 1.f) / L;      // a row that sees nothing is zero
    const float y[4] = {acc.x * f, acc.y * f, acc.z * f, acc.w * f};
    char *dst = p.out + seq * p.out_seq + (int64_t)(h0 + head) * p.out_head;
    store4(dst, ch, p.out_type, y, p.out_inv_step, p.out_zero);
    if (p.lse && ch == 0) p.lse[(int64_t)seq * p.hq + h0 + head] = (M + log2f(L)) * 0.69314718055994530942f;
  }
  if (p.splits > 1) cluster.sync();          // no CTA leaves while another reads its sums
}

// [n_pages][n_heads][page_size][dim] at the cache's strides, boxes of `box` slots of one head: of 128 bytes, 128-byte swizzle, or of
// `dense` channels as they lie. Axes in this order also where heads lie inside slots: a map wants strides that are multiples of 16 below
// 2^40, in any order (heads as the second axis there: 168.6 us instead of 166.4 for 64 ragged sequences).
bool make_cache_map(CUtensorMap *map, const pulpnn_kv_cache_t &c, const void *base, int box, int dense)
{
  sm100::EncodeTiledFn enc = sm100::encode_tiled_fn();
  if (!enc) { set_error(PULPNN_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver"); return false; }
  const bool eight = c.type == PULPNN_TYPE_S8;
  const int size = eight ? 1 : 2;
  const cuuint64_t any = (cuuint64_t)c.head_dim * size;       // the stride of an axis of one element does not matter
  const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.page_size, (cuuint64_t)c.n_heads, (cuuint64_t)c.n_pages};
  const cuuint64_t strides[3] = {c.page_size > 1 ? (cuuint64_t)c.slot_stride * size : any, c.n_heads > 1 ? (cuuint64_t)c.head_stride * size : any,
                                 c.n_pages > 1 ? (cuuint64_t)c.page_stride * size : any};
  const cuuint32_t boxes[4] = {(cuuint32_t)(dense ? dense : eight ? 128 : 64), (cuuint32_t)box, 1, 1}, step[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, eight ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void *>(base), dims, strides,
                         boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE, dense ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { set_error(PULPNN_ERR_CUDA, "cuTensorMapEncodeTiled (cache) failed with code %d", (int)r); return false; }
  return true;
}

struct DecodeLaunch { DecodeProblem &p; const CUtensorMap &k, &v; int64_t pairs, longest; int tile; bool tma; };

// CTAs of a cluster and clusters of a sequence. `slots` CTAs run at a time; `tiles` are a warp's of the longest sequence with one
// CTA. A sequence's time falls with its CTAs and a round of CTAs costs some tiles' time of its own (its first loads and the join:
// 4 us, where a tile of 8 KB takes a slot 0.5 us, memory being shared by all): the number with the least rounds x (share of
// the sequence + 8 tiles), as if all sequences were as long as the table is wide (lengths are not known here). A table wider than the
// sequences takes the most CTAs a sequence: one of 1000 tokens 14.5 us with a table for 131072 (6.9 with one for 1000), 64 of them 75 (51),
// 256 of 300 tokens 105 (59).
void choose_splits(const Context &c, DecodeProblem &p, int64_t pairs, int slots, int64_t longest, int tile)
{
  const int64_t tiles = (longest + WARPS * tile - 1) / (WARPS * tile);
  auto cost = [&](int64_t shares) { return ((pairs * shares + slots - 1) / slots) * ((tiles + shares - 1) / shares + 8); };
  p.splits = 1; p.parts = 1;
  for (int s = 2; s <= MOST_SPLITS; s++)
    if (cost(s) < cost(p.splits)) p.splits = s;
  // more than a cluster: only where these are too few to fill the GPU, and each warp still has 8 tiles (a second kernel costs 3 us)
  if (p.splits == MOST_SPLITS)
    while (pairs * MOST_SPLITS * (p.parts + 1) <= slots && tiles >= (int64_t)MOST_SPLITS * (p.parts + 1) * 8) p.parts++;
  if (c.opt_split_k > 0) {
    p.splits = c.opt_split_k < MOST_SPLITS ? c.opt_split_k : MOST_SPLITS;
    p.parts = c.opt_split_k < 2 * MOST_SPLITS ? 1 : (c.opt_split_k < 512 ? c.opt_split_k / MOST_SPLITS : 64);
  }
}

template <typename T, int DP, int NT, bool EIGHT, bool TMA>
bool decode_go(Context &c, const DecodeLaunch &d)
{
  constexpr int smem = Smem<DP, NT, EIGHT>::BYTES;
  auto k = attn_decode_kernel<T, DP, NT, EIGHT, TMA>;
  static PerDeviceInt resident;
  if (!resident.get(c.device)) {
    if (!cuda_ok(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "cudaFuncSetAttribute(attn_decode)")) return false;
    int n = 0;
    if (!cuda_ok(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k, WARPS * 32, smem), "occupancy(attn_decode)")) return false;
    resident.set(c.device, n < 1 ? 1 : n);
  }
  choose_splits(c, d.p, d.pairs, resident.get(c.device) * c.sm_count, d.longest, d.tile);
  if (d.p.parts > 1) {
    d.p.sums = static_cast<float *>(ctx_stream_alloc(c, (size_t)(d.pairs * d.p.parts) * partial_floats(NT) * 4));
    if (!d.p.sums) d.p.parts = 1;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(d.pairs * d.p.parts * d.p.splits)); cfg.blockDim = dim3(WARPS * 32); cfg.dynamicSmemBytes = smem; cfg.stream = c.stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)d.p.splits; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = d.p.splits > 1 ? 2 : 1;
  bool ok = cuda_ok(cudaLaunchKernelEx(&cfg, k, d.k, d.v, d.p), "pulpnn_attn_decode");
  if (ok) count_launch("attn_decode_kernel");
  if (d.p.parts > 1) {
    if (ok) {
      ok = cuda_ok(launch_pdl(attn_join_kernel<NT>, dim3((unsigned)d.pairs, NT * 8), dim3(MAX_HEAD_DIM), 0, c.stream, d.p), "pulpnn_attn_decode (join)");
      if (ok) count_launch("attn_join_kernel");
    }
    ctx_stream_free(c, d.p.sums);
  }
  return ok;
}
template <typename T, int DP, bool EIGHT>
bool decode_tiles(Context &c, const DecodeLaunch &d)
{
  if (d.p.group > 8) return d.tma ? decode_go<T, DP, 2, EIGHT, true>(c, d) : decode_go<T, DP, 2, EIGHT, false>(c, d);
  return d.tma ? decode_go<T, DP, 1, EIGHT, true>(c, d) : decode_go<T, DP, 1, EIGHT, false>(c, d);
}
template <typename T, bool EIGHT>
bool decode_dim(Context &c, const DecodeLaunch &d)
{
  if (!EIGHT && d.p.dim > 64 && d.p.dim <= 80) return decode_tiles<T, 80, false>(c, d);
  return d.p.dim <= 64 ? decode_tiles<T, 64, EIGHT>(c, d) : (d.p.dim <= 96 ? decode_tiles<T, 96, EIGHT>(c, d) : decode_tiles<T, 128, EIGHT>(c, d));
}

}  // namespace
}  // namespace attn
}  // namespace pulpnn

using namespace pulpnn;
using namespace pulpnn::attn;

extern "C" int pulpnn_attn_decode(const pulpnn_kv_cache_t *cache, const pulpnn_attn_decode_t *a)
{
  const char *who = "pulpnn_attn_decode";
  Context &c = ctx();
  if (const int e = check_cache(who, cache)) return e;
  ATTN_REQUIRE(a && a->n_seqs >= 0, PULPNN_ERR_INVALID_ARG, "%s: %d sequences", who, a ? a->n_seqs : -1);
  if (a->n_seqs == 0) return PULPNN_OK;
  ATTN_REQUIRE(a->q && a->out && a->block_table && a->seq_lens, PULPNN_ERR_INVALID_ARG, "%s: NULL pointer", who);
  ATTN_REQUIRE(is_wide(a->q_type) && (cache->type == PULPNN_TYPE_S8 || cache->type == a->q_type), PULPNN_ERR_UNSUPPORTED,
               "%s: q_type %d with a cache of type %d", who, a->q_type, cache->type);
  ATTN_REQUIRE(a->out_type == a->q_type || a->out_type == PULPNN_TYPE_U8, PULPNN_ERR_UNSUPPORTED, "%s: out_type %d is neither q_type nor U8", who, a->out_type);
  ATTN_REQUIRE(a->n_heads > 0 && a->n_heads % cache->n_heads == 0, PULPNN_ERR_INVALID_ARG, "%s: %d query heads for %d key heads", who,
               a->n_heads, cache->n_heads);
  ATTN_REQUIRE(a->max_pages >= 0 && a->window >= 0, PULPNN_ERR_INVALID_ARG, "%s: max_pages %d, window %d", who, a->max_pages, a->window);
  ATTN_REQUIRE((int64_t)a->max_pages * cache->page_size <= 0x7fff0000, PULPNN_ERR_UNSUPPORTED, "%s: sequences of 2^31 tokens", who);
  if (const int e = check_scale(who, a->scale)) return e;
  if (const int e = check_out(who, a->out_type, a->out_step, a->out_zero)) return e;
  ATTN_REQUIRE(rows_aligned(a->q, 2, {a->q_stride[0], a->q_stride[1]}) &&
               out_aligned(a->out, a->out_type, a->out_stride[0], a->out_stride[1]), PULPNN_ERR_UNSUPPORTED,
               "%s: rows that do not begin on 16-byte boundaries", who);
  ATTN_REQUIRE(aligned(a->block_table, 4) && aligned(a->seq_lens, 4) && aligned(a->lse, 4), PULPNN_ERR_INVALID_ARG, "%s: unaligned table, lengths or lse", who);
  if (!ensure_device(c)) return c.err;
  if (!on_device(c, who, {cache->k, cache->v, cache->k_scale, cache->v_scale, a->q, a->out, a->lse, a->block_table, a->seq_lens})) return c.err;

  DecodeProblem p;
  p.q = static_cast<const char *>(a->q); p.out = static_cast<char *>(a->out); p.lse = a->lse;
  p.table = a->block_table; p.lens = a->seq_lens;
  const int os = type_size(a->out_type);
  p.q_seq = a->q_stride[0] * 2; p.q_head = a->q_stride[1] * 2; p.out_seq = a->out_stride[0] * os; p.out_head = a->out_stride[1] * os;
  p.table_stride = a->table_stride;
  p.cache = view_of(*cache);
  p.hq = a->n_heads; p.group = a->n_heads / cache->n_heads; p.dim = cache->head_dim; p.max_pages = a->max_pages; p.window = a->window;
  p.q_type = a->q_type; p.out_type = a->out_type;
  p.scale_log2 = a->scale * 1.4426950408889634074f;
  p.out_inv_step = a->out_type == PULPNN_TYPE_U8 ? 1.f / a->out_step : 1.f; p.out_zero = a->out_zero;
  const bool two = p.group > 8, eight = cache->type == PULPNN_TYPE_S8;
  p.head_tiles = (p.group + (two ? 15 : 7)) / (two ? 16 : 8);
  const int64_t pairs = (int64_t)a->n_seqs * cache->n_heads * p.head_tiles;
  ATTN_REQUIRE(pairs <= 0x0fffffff, PULPNN_ERR_UNSUPPORTED, "%s: %d sequences of %d heads", who, a->n_seqs, a->n_heads);
  int64_t longest = (int64_t)a->max_pages * cache->page_size;
  if (a->window > 0 && a->window < longest) longest = a->window;
  const int tile = eight || p.dim <= 64 ? 32 : 16;
  // pages that hold whole runs of 16 tokens come by TMA, whose maps want positive strides below 2^40 bytes
  auto fits = [&](int n, int64_t s) { return n == 1 || (s > 0 && s < (int64_t)1 << 38); };
  const bool tma = cache->page_size % 16 == 0 && fits(cache->page_size, cache->slot_stride) && fits(cache->n_heads, cache->head_stride) &&
                   fits(cache->n_pages, cache->page_stride);
  p.box = tile == 32 && cache->page_size % 32 == 0 && p.window == 0 ? 32 : 16;
  CUtensorMap mk, mv;
  p.status = nullptr; p.sums = nullptr;
  if (tma) {
    if (!ctx_status_word_unless_capturing(c, &p.status)) return c.err;
    const int dense = !eight && p.dim > 64 && p.dim <= 80 ? 80 : 0;
    if (!make_cache_map(&mk, *cache, cache->k, p.box, dense) || !make_cache_map(&mv, *cache, cache->v, p.box, dense)) return c.err;
  }
  const DecodeLaunch d = {p, mk, mv, pairs, longest, tile, tma};
  const bool ok = eight ? decode_dim<__half, true>(c, d)
                        : (a->q_type == PULPNN_TYPE_F16 ? decode_dim<__half, false>(c, d) : decode_dim<__nv_bfloat16, false>(c, d));
  return ok ? PULPNN_OK : c.err;
}
