// attn_prompt.cu -- pulpnn_attn_prompt: attention over whole prompts, on tcgen05.
//
//   O = softmax(scale * Q K^T, masked) V   per sequence and query head, in tiles of 128 queries x 128 keys.
//
// A CTA holds two tiles of queries ("units") and walks over the keys that either sees; both multiply with every K and V
// tile it loads. The units of a key head are its 128-row tiles times the G query heads that share it, heads
// fastest, and a CTA takes two that follow one another: two heads of the same rows where G > 1 (the same causal
// range, and both busy however short the sequence is), two neighbouring row tiles where G = 1.
//
//   warps 0-3, 4-7  softmax of unit 0 and 1: a thread is a row. S comes from TMEM, the weights go back there as the 16-bit
//                   operand of the second product, in the columns S had.
//   warp 8          loads Q, then K and V tiles in turn, by TMA into a ring of stages
//   warp 9          issues the MMAs: S = Q K^T (both from shared memory), O += P V (P from TMEM). While one unit's weights
//                   are computed, the other unit's products run.
//   warps 10, 11    guard the V tiles in which some query of the CTA does not see some key: a weight of 0 does
//                   not keep an infinity or a NaN out of a sum of products, so rows behind the sequence's end (another sequence's)
//                   become 0, and so do infinities and NaN among the rest, which the epilogue then adds to
//                   the rows that do see them.
//
// TMEM: S of unit 0 and 1 (128 columns each), O of unit 0 and 1 (64 or 128 each).
// The running maximum is a reference that has to be near the true one only: it is raised, and O rescaled in TMEM by
// the softmax warps themselves, when a score is more than 2^LAG above it, which after the first tiles is rare.
// Between the commit that announces S(j) and its own arrival with P(j), a softmax group has O to itself: the
// commit comes behind the MMAs of tile j - 1.
#include "attention.cuh"
#include "sm100_primitives.cuh"

namespace pulpnn {
namespace attn {
namespace {

using namespace sm100;

constexpr int BQ = 128, BK = 128, THREADS = 384;
constexpr int WARP_LOAD = 8, WARP_MMA = 9, WARP_GUARD = 10, GUARD_THREADS = 64;
constexpr float LAG = 8.f, NOTHING = -1e30f;
enum { ST_LOAD = 1 << 20, ST_MMA = 1 << 21, ST_SOFTMAX = 1 << 22, ST_GUARD = 1 << 23, ST_EPI = 1 << 24 };

struct PromptProblem {
  const char *v;
  char *out;
  float *lse;
  const int *cu_q, *cu_k;
  int64_t v_row, v_head, out_row, out_head;       // bytes
  int nq, nk, seqs, hq, group, dim, causal, window, out_type, out_zero;
  float scale_log2, out_inv_step;
  int *status;
};

template <int DP> struct Shape {
  static constexpr int BOXES = DP / 64;                        // of 64 channels: rows of 128 bytes, swizzled
  static constexpr int BOX = 128 * 128;                        // bytes
  static constexpr int TILE = BOXES * BOX;
  static constexpr int STAGES = DP == 128 ? 4 : 8;             // even: keys in the even stages, values in the odd ones
  static constexpr int SMEM = (2 + STAGES) * TILE + 1024 /* barriers */ + 1024 /* alignment */;
};

struct Control {
  uint64_t q_full[2], kv_full[8], kv_empty[8], clean[4], s_full[2], p_full[2], drain;
  uint32_t tmem;
  int abort_flag, dirty;
  int warp_total[THREADS / 32];
  int found, q0, k0, lq, lk, pair;
};

// D(tmem) (+)= A(smem) * B(smem)^T and A(tmem) * B(smem), 16-bit operands, 32-bit sums
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add)
{
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add ? 1 : 0) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add)
{
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add ? 1 : 0) : "memory");
}
// V as it lies, keys x channels: the product's N (channels) is contiguous. Blocks of 64 channels are a box apart
// (leading offset), groups of 8 keys 1024 bytes (stride offset).
__device__ __forceinline__ uint64_t desc_v(uint32_t saddr)
{
  return (uint64_t)((saddr & 0x3ffffu) >> 4) | (uint64_t)((128 * 128) >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
// D = f32 (1 at bit 4), types of A and B (0 = f16, 1 = bf16) at bits 7 and 10, bit 16: B's N contiguous, N / 8, M / 16
__device__ __forceinline__ uint32_t idesc16(bool bf16, bool b_n_major, int n)
{
  return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (b_n_major ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
}
__device__ __forceinline__ void tmem_ld_16(uint32_t taddr, uint32_t (&r)[16])
{
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t (&r)[16])
{
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
               ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x)
{
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T> struct Kind;
template <> struct Kind<__half> { static constexpr bool BF16 = false; static constexpr unsigned EXP = 0x7c00u; };
template <> struct Kind<__nv_bfloat16> { static constexpr bool BF16 = true; static constexpr unsigned EXP = 0x7f80u; };

// A tile of queries: rows row0 .. row0 + rows - 1 of head `head`, the first at position pos; it sees the key tiles lo .. hi - 1.
struct Unit { int row0, rows, head, pos, lo, hi, keys; };

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, 1)
attn_prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const PromptProblem p)
{
  using SH = Shape<DP>;
  extern __shared__ char raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  char *smem = raw + (base - smem_u32(raw));
  const uint32_t s_q = base, s_kv = base + 2 * SH::TILE;
  Control &ct = *reinterpret_cast<Control *>(smem + (2 + SH::STAGES) * SH::TILE);
  static_assert(sizeof(Control) <= 1024, "control block");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int *abort_flag = &ct.abort_flag;

  if (threadIdx.x == 0) {
    ct.abort_flag = 0; ct.dirty = 0; ct.found = 0;
    for (int x = 0; x < 2; x++) { mbar_init(&ct.q_full[x], 1); mbar_init(&ct.s_full[x], 1); mbar_init(&ct.p_full[x], 4); }
    for (int s = 0; s < SH::STAGES; s++) { mbar_init(&ct.kv_full[s], 1); mbar_init(&ct.kv_empty[s], 1); }
    for (int s = 0; s < SH::STAGES / 2; s++) mbar_init(&ct.clean[s], 2);
    mbar_init(&ct.drain, 1);
    mbar_fence_init();
  }
  pdl_wait();
  // ---- which two units: the sequence whose pairs of units hold number blockIdx.x ----
  {
    int before = 0;
    __syncthreads();
    for (int s0 = 0; s0 < p.seqs; s0 += THREADS) {
      const int b = s0 + threadIdx.x;
      int count = 0, q0 = 0, lq = 0;
      if (b < p.seqs) {
        q0 = min(max(__ldg(p.cu_q + b), 0), p.nq);
        lq = min(max(__ldg(p.cu_q + b + 1), q0), p.nq) - q0;
        count = (int)(((int64_t)((lq + BQ - 1) / BQ) * p.group + 1) / 2);
      }
      int incl = count;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int y = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += y;
      }
      if (lane == 31) ct.warp_total[warp] = incl;
      __syncthreads();
      int total = 0, off = before;
      for (int w = 0; w < THREADS / 32; w++) { if (w < warp) off += ct.warp_total[w]; total += ct.warp_total[w]; }
      const int at = (int)blockIdx.x - (off + incl - count);
      if (at >= 0 && at < count) {
        const int k0 = min(max(__ldg(p.cu_k + b), 0), p.nk);
        ct.q0 = q0; ct.lq = lq; ct.k0 = k0; ct.lk = min(max(__ldg(p.cu_k + b + 1), k0), p.nk) - k0;
        ct.pair = count - 1 - at;          // the last rows of a causal sequence see the most keys: they begin first
        ct.found = 1;
      }
      before += total;
      __syncthreads();
      if (ct.found) break;
    }
  }
  if (!ct.found) return;
  if (warp == WARP_MMA) tmem_alloc(&ct.tmem, 512);
  const int q0 = ct.q0, k0 = ct.k0, lq = ct.lq, lk = ct.lk, kvh = blockIdx.y;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ct.tmem;

  Unit un[2];
#pragma unroll
  for (int x = 0; x < 2; x++) {
    const int u = 2 * ct.pair + x, rt = u / p.group;
    Unit &w = un[x];
    w.row0 = rt * BQ; w.head = kvh * p.group + u - rt * p.group;
    w.rows = min(max(lq - w.row0, 0), BQ);
    w.pos = w.row0 + lk - lq;
    w.keys = w.rows == 0 ? 0 : (p.causal ? min(lk, max(w.pos + w.rows, 0)) : lk);       // it sees none from here on
    const int from = p.window > 0 ? max(0, w.pos - p.window + 1) : 0;
    w.lo = from / BK; w.hi = (w.keys + BK - 1) / BK;
    if (from >= w.keys) w.lo = w.hi = 0;
  }
  const bool any0 = un[0].hi > un[0].lo, any1 = un[1].hi > un[1].lo;
  const int lo = !any0 ? un[1].lo : (!any1 ? un[0].lo : min(un[0].lo, un[1].lo)), hi = max(un[0].hi, un[1].hi);
  auto sees = [](const Unit &u, int j) { return j >= u.lo && j < u.hi; };
  // whether some row of the unit does not see some key of tile j
  auto masked = [&](const Unit &u, int j) {
    const int k = j * BK, end = p.causal ? min(lk, u.pos + 1) : lk;
    return k + BK > end || (p.window > 0 && k < u.pos + u.rows - p.window);
  };
  auto guarded = [&](int j) { return (sees(un[0], j) && masked(un[0], j)) || (sees(un[1], j) && masked(un[1], j)); };

  if (warp >= WARP_LOAD) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == WARP_LOAD) {
      if (lane == 0) {
        int issued = 0;
        bool ok = true;
#pragma unroll
        for (int x = 0; x < 2; x++) {
          if (un[x].hi <= un[x].lo) continue;
          mbar_arrive_expect_tx(&ct.q_full[x], SH::TILE);
          for (int b = 0; b < SH::BOXES; b++)
            tma_load_3d(smem + x * SH::TILE + b * SH::BOX, &map_q, &ct.q_full[x], b * 64, un[x].head, q0 + un[x].row0);
        }
        for (int e = 0; e < 2 * (hi - lo) && ok; e++) {
          const int st = e % SH::STAGES, j = lo + (e >> 1);
          if (!(ok = mbar_wait(&ct.kv_empty[st], ((e / SH::STAGES) & 1) ^ 1, abort_flag, p.status, ST_LOAD))) break;
          mbar_arrive_expect_tx(&ct.kv_full[st], SH::TILE);
          for (int b = 0; b < SH::BOXES; b++)
            tma_load_3d(smem + (2 + st) * SH::TILE + b * SH::BOX, e & 1 ? &map_v : &map_k, &ct.kv_full[st], b * 64, kvh, k0 + j * BK);
          issued = e + 1;
        }
        if (!ok) {        // given up: the copies in flight must land before the CTA's shared memory is given away
          volatile int never = 0;
#pragma unroll
          for (int x = 0; x < 2; x++)
            if (un[x].hi > un[x].lo) mbar_wait(&ct.q_full[x], 0, &never, nullptr, 0);
          for (int e = max(0, issued - SH::STAGES); e < issued; e++)
            mbar_wait(&ct.kv_full[e % SH::STAGES], (e / SH::STAGES) & 1, &never, nullptr, 0);
        }
      }
    } else if (warp == WARP_MMA) {
      if (lane == 0) {
        const int ksteps = (p.dim + 15) / 16;
        const uint32_t id_s = idesc16(Kind<T>::BF16, false, BK), id_o = idesc16(Kind<T>::BF16, true, ksteps * 16);
        int pcount[2] = {0, 0};
        bool ok = true, have_q[2] = {false, false};
        auto issue_s = [&](int x, int j) {      // the caller has waited for K(j)
          if (!have_q[x]) { have_q[x] = true; if (!(ok = mbar_wait(&ct.q_full[x], 0, abort_flag, p.status, ST_MMA))) return; }
          const uint32_t a = s_q + x * SH::TILE, b = s_kv + ((2 * (j - lo)) % SH::STAGES) * SH::TILE;
          tc_fence_after();
          for (int ks = 0; ks < ksteps; ks++) {
            const uint32_t off = (ks >> 2) * SH::BOX + (ks & 3) * 32;
            umma_ss(tmem + x * 128, umma_smem_desc<128>(a + off), umma_smem_desc<128>(b + off), id_s, ks > 0);
          }
          umma_commit(&ct.s_full[x]);
        };
        auto wait_kv = [&](int e) { return mbar_wait(&ct.kv_full[e % SH::STAGES], (e / SH::STAGES) & 1, abort_flag, p.status, ST_MMA); };
        if (lo < hi) {
          ok = wait_kv(0);
#pragma unroll
          for (int x = 0; x < 2; x++)
            if (ok && sees(un[x], lo)) issue_s(x, lo);
          if (ok) umma_commit(&ct.kv_empty[0]);
        }
        for (int j = lo; j < hi && ok; j++) {
          const int ev = 2 * (j - lo) + 1, ek = ev + 1;
          bool have_v = false, have_k = false;
#pragma unroll
          for (int x = 0; x < 2; x++) {
            if (ok && sees(un[x], j)) {
              if (!have_v) {
                have_v = true;
                ok = wait_kv(ev) && mbar_wait(&ct.clean[(ev % SH::STAGES) >> 1], (ev / SH::STAGES) & 1, abort_flag, p.status, ST_MMA);
                if (!ok) break;
              }
              if (!(ok = mbar_wait(&ct.p_full[x], pcount[x] & 1, abort_flag, p.status, ST_MMA))) break;
              pcount[x]++;
              tc_fence_after();
              const uint32_t b = s_kv + (ev % SH::STAGES) * SH::TILE;
              const int parts = min(BK / 16, (un[x].keys - j * BK + 15) / 16);      // keys that none of its rows sees are left out
              for (int kk = 0; kk < parts; kk++)
                umma_ts(tmem + 256 + x * DP, tmem + x * 128 + kk * 8, desc_v(b + kk * 2048), id_o, j > un[x].lo || kk > 0);
            }
            if (ok && sees(un[x], j + 1)) {
              if (!have_k) { have_k = true; if (!(ok = wait_kv(ek))) break; }
              issue_s(x, j + 1);
            } else if (ok && sees(un[x], j)) {
              umma_commit(&ct.s_full[x]);         // O is complete
            }
          }
          if (!ok) break;
          umma_commit(&ct.kv_empty[ev % SH::STAGES]);
          if (j + 1 < hi) umma_commit(&ct.kv_empty[ek % SH::STAGES]);
        }
        if (!ok) {        // given up: the MMAs in flight must end before TMEM is given back
          volatile int never = 0;
          umma_commit(&ct.drain);
          mbar_wait(&ct.drain, 0, &never, nullptr, 0);
        }
      }
    } else {
      const int id = threadIdx.x - WARP_GUARD * 32;
      for (int j = lo; j < hi; j++) {
        const int e = 2 * (j - lo) + 1, st = e % SH::STAGES;
        if (!mbar_wait(&ct.kv_full[st], (e / SH::STAGES) & 1, abort_flag, p.status, ST_GUARD)) break;
        if (guarded(j)) {
          const int rows = lk - j * BK;
          bool odd = false;
          for (int i = id; i < SH::TILE / 16; i += GUARD_THREADS) {
            uint4 *at = reinterpret_cast<uint4 *>(smem + (2 + st) * SH::TILE) + i;
            if (((i >> 3) & 127) >= rows) { *at = make_uint4(0, 0, 0, 0); continue; }
            const uint4 w = *at;
            constexpr unsigned E = Kind<T>::EXP;
            // the exponent's bits all set: adding one at their lowest place carries into the sign's
            auto bad = [](unsigned v) { return ((v & (E * 0x10001u)) + (E & (~E + 1u)) * 0x10001u) & 0x80008000u; };
            const unsigned x = bad(w.x), y = bad(w.y), z = bad(w.z), t = bad(w.w);
            if (x | y | z | t) {
              auto keep = [](unsigned v, unsigned b) { return v & ~((b >> 15) * 0xffffu); };
              *at = make_uint4(keep(w.x, x), keep(w.y, y), keep(w.z, z), keep(w.w, t));
              odd = true;
            }
          }
          if (odd) *reinterpret_cast<volatile int *>(&ct.dirty) = 1;
          fence_proxy_async();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ct.clean[st >> 1]);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int x = warp >> 2, r = threadIdx.x & 127;
    const Unit w = x == 0 ? un[0] : un[1];
    const uint32_t rowbase = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_s = rowbase + x * 128, t_o = rowbase + 256 + x * DP;
    const int pos = w.pos + r;
    const int last = p.causal ? min(lk - 1, pos) : lk - 1, first = p.window > 0 ? pos - p.window + 1 : 0;
    const int cols = (p.dim + 15) / 16;
    float m = NOTHING, l = 0.f;
    bool ok = true;
    uint32_t phase = 0;
    for (int j = w.lo; j < w.hi; j++) {
      if (!(ok = mbar_wait(&ct.s_full[x], phase, abort_flag, p.status, ST_SOFTMAX))) break;
      phase ^= 1;
      tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int i = 0; i < 4; i++) tmem_ld_32(t_s + i * 32, s[i]);
      tmem_wait_ld();
      if (masked(w, j)) {
        const int a = first - j * BK, b = last - j * BK;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int c = 0; c < 32; c++)
            if (i * 32 + c < a || i * 32 + c > b) s[i][c] = 0xff800000u;
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 32; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) top[i] = fmaxf(top[i], __uint_as_float(s[i][c]));
      const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.scale_log2;
      if (__any_sync(0xffffffffu, most > m + LAG)) {
        const float to = fmaxf(m, most), f = ex2(m - to);
        m = to;
        l *= f;
        if (j > w.lo) {
          for (int c = 0; c < cols; c++) {
            uint32_t o[16];
            tmem_ld_16(t_o + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st_16(t_o + c * 16, o);
          }
        }
      }
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        uint32_t w16[16];
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          const float e0 = ex2(fmaf(__uint_as_float(s[i][c]), p.scale_log2, -m)), e1 = ex2(fmaf(__uint_as_float(s[i][c + 1]), p.scale_log2, -m));
          sum[i] += e0 + e1;
          w16[c / 2] = pack2<T>(e0, e1);       // off by 2^-8 (bf16) or 2^-11 (fp16) of each weight at most; their sum is taken unrounded
        }
        tmem_st_16(t_s + i * 16, w16);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ct.p_full[x]);
    }
    // ---- epilogue ----
    const bool any = w.hi > w.lo;
    if (ok && any) ok = mbar_wait(&ct.s_full[x], phase, abort_flag, p.status, ST_EPI);
    if (ok) {
      tc_fence_after();
      const bool live = r < w.rows;
      const int64_t row = q0 + w.row0 + r;
      const float inv = l == 0.f ? 0.f : 1.f / l;         // a row that sees nothing is zero
      char *dst = p.out + row * p.out_row + (int64_t)w.head * p.out_head;
      const bool dirty = any && *reinterpret_cast<volatile int *>(&ct.dirty);
      for (int c = 0; c < cols; c++) {
        float y[16];
        if (any) {
          uint32_t o[16];
          tmem_ld_16(t_o + c * 16, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; i++) y[i] = inv == 0.f ? 0.f : __uint_as_float(o[i]) * inv;
        } else {
#pragma unroll
          for (int i = 0; i < 16; i++) y[i] = 0.f;
        }
        if (dirty && live) {      // the infinities and NaN that the guards took out of the tiles, where this row sees them
          for (int j = w.lo; j < w.hi; j++) {
            if (!guarded(j)) continue;
            for (int k = max(first, j * BK); k <= min(last, j * BK + BK - 1); k++) {
              const T *v = reinterpret_cast<const T *>(p.v + (int64_t)(k0 + k) * p.v_row + (int64_t)kvh * p.v_head) + c * 16;
#pragma unroll
              for (int i = 0; i < 16; i++)
                if (c * 16 + i < p.dim) {
                  const float z = (float)v[i];
                  if (!(fabsf(z) <= 3.402823466e38f)) y[i] += z;
                }
            }
          }
        }
        if (live) {
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            if (c * 16 + i < p.dim) {
              const float z[4] = {y[i], y[i + 1], y[i + 2], y[i + 3]};
              store4(dst, c * 16 + i, p.out_type, z, p.out_inv_step, p.out_zero);
            }
        }
      }
      if (live && p.lse) p.lse[row * p.hq + w.head] = (m + log2f(l)) * 0.69314718055994530942f;
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == WARP_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// [rows][heads][dim] of 16-bit values; boxes of 64 channels x 1 head x 128 rows, 128-byte swizzle. Channels and rows
// outside read as zero.
bool make_rows_map(CUtensorMap *map, int type, const void *p, int rows, int heads, int dim, const int64_t *stride)
{
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) { set_error(PULPNN_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver"); return false; }
  const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)rows};
  // the stride of an axis of one element does not matter, and may be anything
  const cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? stride[1] * 2 : dim * 2), (cuuint64_t)(rows > 1 ? stride[0] * 2 : dim * 2)};
  const cuuint32_t box[3] = {64, 1, 128}, step[3] = {1, 1, 1};
  const CUresult r = enc(map, type == PULPNN_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                         const_cast<void *>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { set_error(PULPNN_ERR_CUDA, "cuTensorMapEncodeTiled (rows) failed with code %d", (int)r); return false; }
  return true;
}

template <typename T, int DP>
bool prompt_go(Context &c, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, const PromptProblem &p, dim3 grid)
{
  auto k = attn_prompt_kernel<T, DP>;
  static PerDeviceInt ready;
  if (!ready.get(c.device)) {
    if (!cuda_ok(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DP>::SMEM), "cudaFuncSetAttribute(attn_prompt)")) return false;
    ready.set(c.device, 1);
  }
  if (!cuda_ok(launch_pdl(k, grid, dim3(THREADS), Shape<DP>::SMEM, c.stream, mq, mk, mv, p), "pulpnn_attn_prompt")) return false;
  count_launch("attn_prompt_kernel");
  return true;
}

}  // namespace
}  // namespace attn
}  // namespace pulpnn

using namespace pulpnn;
using namespace pulpnn::attn;

extern "C" int pulpnn_attn_prompt(const pulpnn_attn_prompt_t *a)
{
  const char *who = "pulpnn_attn_prompt";
  Context &c = ctx();
  ATTN_REQUIRE(a && a->n_q_rows >= 0 && a->n_k_rows >= 0 && a->n_seqs >= 0, PULPNN_ERR_INVALID_ARG, "%s: %d and %d rows, %d sequences", who,
               a ? a->n_q_rows : -1, a ? a->n_k_rows : -1, a ? a->n_seqs : -1);
  if (a->n_q_rows == 0 || a->n_seqs == 0) return PULPNN_OK;
  ATTN_REQUIRE(a->q && a->out && a->cu_q && a->cu_k && (a->n_k_rows == 0 || (a->k && a->v)), PULPNN_ERR_INVALID_ARG, "%s: NULL pointer", who);
  ATTN_REQUIRE(is_wide(a->type), PULPNN_ERR_UNSUPPORTED, "%s: type %d", who, a->type);
  ATTN_REQUIRE(a->out_type == a->type || a->out_type == PULPNN_TYPE_U8, PULPNN_ERR_UNSUPPORTED, "%s: out_type %d is neither the inputs' nor U8", who, a->out_type);
  ATTN_REQUIRE(a->n_kv_heads > 0 && a->n_heads > 0 && a->n_heads % a->n_kv_heads == 0 && a->n_heads <= 65535, PULPNN_ERR_INVALID_ARG,
               "%s: %d query heads for %d key heads", who, a->n_heads, a->n_kv_heads);
  ATTN_REQUIRE(a->head_dim > 0 && a->head_dim <= MAX_HEAD_DIM && a->head_dim % 8 == 0, PULPNN_ERR_UNSUPPORTED,
               "%s: head_dim %d is not a multiple of 8 up to %d", who, a->head_dim, MAX_HEAD_DIM);
  ATTN_REQUIRE(a->n_q_rows <= 0x3fffffff && a->n_k_rows <= 0x3fffffff, PULPNN_ERR_UNSUPPORTED, "%s: 2^30 rows or more", who);
  ATTN_REQUIRE(a->window >= 0 && (a->window == 0 || a->causal), PULPNN_ERR_INVALID_ARG, "%s: window %d%s", who, a->window, a->causal ? "" : " of a call that is not causal");
  if (const int e = check_scale(who, a->scale)) return e;
  if (const int e = check_out(who, a->out_type, a->out_step, a->out_zero)) return e;
  ATTN_REQUIRE(rows_aligned(a->q, 2, {a->q_stride[0], a->q_stride[1]}) && rows_aligned(a->k, 2, {a->k_stride[0], a->k_stride[1]}) &&
               rows_aligned(a->v, 2, {a->v_stride[0], a->v_stride[1]}) &&
               out_aligned(a->out, a->out_type, a->out_stride[0], a->out_stride[1]), PULPNN_ERR_UNSUPPORTED,
               "%s: rows that do not begin on 16-byte boundaries", who);
  const int64_t *strides[3] = {a->q_stride, a->k_stride, a->v_stride};
  for (int i = 0; i < 3; i++)
    ATTN_REQUIRE(((i == 0 ? a->n_q_rows : a->n_k_rows) <= 1 || (strides[i][0] > 0 && strides[i][0] < (int64_t)1 << 38)) &&
                 ((i == 0 ? a->n_heads : a->n_kv_heads) <= 1 || (strides[i][1] > 0 && strides[i][1] < (int64_t)1 << 38)),
                 PULPNN_ERR_UNSUPPORTED, "%s: strides that are not positive, or 2^38 and more", who);
  ATTN_REQUIRE(aligned(a->cu_q, 4) && aligned(a->cu_k, 4) && aligned(a->lse, 4), PULPNN_ERR_INVALID_ARG, "%s: unaligned offsets or lse", who);
  if (!ensure_device(c)) return c.err;
  if (!on_device(c, who, {a->q, a->k, a->v, a->out, a->lse, a->cu_q, a->cu_k})) return c.err;

  PromptProblem p;
  const int os = type_size(a->out_type);
  p.v = static_cast<const char *>(a->v); p.out = static_cast<char *>(a->out); p.lse = a->lse; p.cu_q = a->cu_q; p.cu_k = a->cu_k;
  p.v_row = a->v_stride[0] * 2; p.v_head = a->v_stride[1] * 2; p.out_row = a->out_stride[0] * os; p.out_head = a->out_stride[1] * os;
  p.nq = a->n_q_rows; p.nk = a->n_k_rows; p.seqs = a->n_seqs; p.hq = a->n_heads; p.group = a->n_heads / a->n_kv_heads; p.dim = a->head_dim;
  p.causal = a->causal != 0; p.out_type = a->out_type; p.out_zero = a->out_zero;
  p.window = a->window < 0x3fffffff ? a->window : 0x3fffffff;      // positions are below 2^30
  p.scale_log2 = a->scale * 1.4426950408889634074f;
  p.out_inv_step = a->out_type == PULPNN_TYPE_U8 ? 1.f / a->out_step : 1.f;
  if (!ctx_status_word_unless_capturing(c, &p.status)) return c.err;
  // without keys there is nothing to load, but the maps want an address
  const void *k = a->n_k_rows ? a->k : a->q, *v = a->n_k_rows ? a->v : a->q;
  CUtensorMap mq, mk, mv;
  if (!make_rows_map(&mq, a->type, a->q, a->n_q_rows, a->n_heads, a->head_dim, a->q_stride)) return c.err;
  if (a->n_k_rows) {
    if (!make_rows_map(&mk, a->type, k, a->n_k_rows, a->n_kv_heads, a->head_dim, a->k_stride) ||
        !make_rows_map(&mv, a->type, v, a->n_k_rows, a->n_kv_heads, a->head_dim, a->v_stride)) return c.err;
  } else {
    mk = mv = mq;
  }
  // at most this many pairs of units: a sequence's rows fill all its tiles but one, and a pair may be half empty
  const int64_t pairs = (((int64_t)a->n_q_rows / BQ + a->n_seqs) * p.group + a->n_seqs + 1) / 2;
  ATTN_REQUIRE(pairs <= 0x7fffffff, PULPNN_ERR_UNSUPPORTED, "%s: %d rows in %d sequences", who, a->n_q_rows, a->n_seqs);
  const dim3 grid((unsigned)pairs, (unsigned)a->n_kv_heads);
  const bool f16 = a->type == PULPNN_TYPE_F16, narrow = a->head_dim <= 64;
  const bool ok = f16 ? (narrow ? prompt_go<__half, 64>(c, mq, mk, mv, p, grid) : prompt_go<__half, 128>(c, mq, mk, mv, p, grid))
                      : (narrow ? prompt_go<__nv_bfloat16, 64>(c, mq, mk, mv, p, grid) : prompt_go<__nv_bfloat16, 128>(c, mq, mk, mv, p, grid));
  return ok ? PULPNN_OK : c.err;
}
