// attn_prompt.cu -- pulpnn_attn_prompt: attention over whole prompts, on tcgen05.
//
//   O = softmax(scale * Q K^T, masked) V   per sequence and query head, in tiles of 128 queries x 128 keys.
//
// Work comes in items of two tiles of queries ("units"), which walk together over the keys that either sees; both
// multiply with every K and V tile that is loaded. The units of a key head are its 128-row tiles times the G query heads
// that share it, heads fastest, and an item is two that follow one another: two heads of the same rows where G > 1 (the
// same causal range, and both busy however short the sequence is), two neighbouring row tiles where G = 1.
//
// One CTA an SM. It begins with the item of its own block index and takes further ones from blocks that have not
// started yet (clusterlaunchcontrol), so that nothing is set up twice and no SM waits at the end of a fixed share; a
// sequence's last rows, which see the most keys, come first. Where there are no more units than SMs, each is an item.
//
//   warps 0-3, 4-7  softmax of unit 0 and 1: a thread is a row. S comes from TMEM, the weights go back there as the 16-bit
//                   operand of the second product. At an item's end they also write its rows.
//   warp 8          loads Q, then K and V tiles in turn, by TMA into a ring of stages
//   warp 9          issues the MMAs: S = Q K^T (both from shared memory), O += P V (P from TMEM). While one unit's weights
//                   are computed, the other unit's products run; an item's first S follow the last O of the one before.
//   warps 10, 11    guard the V tiles in which some query of the item does not see some key: a weight of 0 does
//                   not keep an infinity or a NaN out of a sum of products, so rows behind the sequence's end (another
//                   sequence's) become 0, and so do infinities and NaN among the rest, which the epilogue then adds to
//                   the rows that do see them. Warp 10 also fetches the items, one ahead.
//
// What bounds it: 128 keys of two units take the tensor cores 2048 (1024) cycles at 128 (64) channels, and the special
// function units, 16 exponentials a cycle, 2048 cycles at any number of channels. What decides is therefore how much of a
// unit's cycle S -> weights -> P V -> S is in the way of its own next step:
//   64 channels: TMEM (512 columns) holds S, P and O of both units side by side. S of the next tile is computed as soon as
//     the softmax warps have S in registers, and they never wait for it.
//   128 channels: P has to lie in columns that S had, and the next S comes behind P V. The weights are handed over in two
//     halves, so that the first half's product runs under the second half's exponentials.
// The running maximum is a reference that has to be near the true one only: it is taken from an item's first tile, and raised
// (O being rescaled in TMEM by the softmax warps themselves) when a weight comes out above 2^15, which is rare. fp16 ends at
// 2^-24 on the other side, and many small weights make a sum: there the reference lies 2^UNDER below the maximum when it is set, so that
// each weight is off by 2^-30 of the largest one at most. (128 weights of a tile that all are the largest come to 2^12.)
//
// Measured (one B200): 16384 causal tokens, 32 query and 8 key heads of 128 channels in bf16, 2000 us (1100 of the 1670 TFLOP/s
// that a plain matrix product reaches), up to 2085 in a long run, where the power limit lowers the clock to 1665 of 1965 MHz; of 8192 tokens
// the tensor cores and the special function units are busy for 62 % of the cycles each. 24 packed prompts of 28 heads of 64
// channels 210 us, where the exponentials alone take 82 and the matrix products 57; 300 tokens 11.2 us: the set-up, three
// key tiles one after the other and the epilogue.
#include "attention.cuh"
#include "sm100_primitives.cuh"

namespace pulpnn {
namespace attn {
namespace {

using namespace sm100;

constexpr int BQ = 128, BK = 128, THREADS = 384;
constexpr int WARP_LOAD = 8, WARP_MMA = 9, WARP_GUARD = 10, GUARD_THREADS = 64;
constexpr float NOTHING = -3.402823466e38f;       // the lowest number: any score is at least that
enum { ST_LOAD = 1 << 20, ST_MMA = 1 << 21, ST_SOFTMAX = 1 << 22, ST_GUARD = 1 << 23, ST_EPI = 1 << 24 };

struct PromptProblem {
  const char *v;
  char *out;
  float *lse;
  const int *cu_q, *cu_k;
  int64_t v_row, v_head, out_row, out_head;       // bytes
  FastDiv by_group;
  int units;                                      // of an item: 2, or 1 where all of them find an SM at once
  int merged;                                     // items come longest first
  int nq, nk, seqs, hq, group, dim, causal, window, out_type, out_zero;
  float scale_log2, out_inv_step;
  int *status;
};

template <int DP> struct Shape {
  static constexpr int BOXES = DP / 64;                        // of 64 channels: rows of 128 bytes, swizzled
  static constexpr int BOX = 128 * 128;                        // bytes
  static constexpr int TILE = BOXES * BOX;
  // TMEM: S of unit 0 and 1, O of unit 0 and 1, and P of both where there is room
  static constexpr bool APART = DP == 64;
  static constexpr int O_AT = 256, P_AT = APART ? 256 + 2 * DP : 0, P_STEP = APART ? 64 : 128;
  static constexpr int STAGES = DP == 128 ? 4 : 8;             // even: keys in the even stages, values in the odd ones
  static constexpr int STAGING = 32 * 128;                     // of a softmax warp: 32 rows of 64 channels on their way out
  static constexpr int SMEM = (2 + STAGES) * TILE + 1024 /* barriers */ + 8 * STAGING + 1024 /* alignment */;
};

// A tile of queries: rows row0 .. row0 + rows - 1 of head `head`, the first at position pos; it sees the key tiles lo .. hi - 1.
struct Unit { int row0, rows, head, pos, lo, hi; };
// An item's units and the key tiles lo .. hi - 1 that either sees.
struct Work { Unit u[2]; int q0, k0, lk, kvh, lo, hi; };
struct Item { Work w; int end, dirty; };
constexpr int ITEMS = 3;

struct Control {
  uint64_t q_full[2], q_empty[2], kv_full[8], kv_empty[8], clean[4], s_full[2], s_free[2], p_half[2], p_full[2], pv_done[2], o_full[2], item_full[ITEMS], item_empty[ITEMS], next, drain;
  uint4 answer;                    // to the request for another block's work
  Item item[ITEMS];
  uint32_t tmem;
  int abort_flag;
};

// The work of a block that has not started: asks for it, and reads the answer (false: there is none left).
__device__ __forceinline__ void ask_for_block(uint4 *answer, uint64_t *bar)
{
  mbar_arrive_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool block_of(const uint4 *answer, int &x, int &y)
{
  uint32_t got, bx, by;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t.reg .b32 z;\n\t"
      "ld.shared.b128 r, [%3];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, %2, z, _}, r;\n\t}"
      : "=&r"(got), "=&r"(bx), "=&r"(by) : "r"(smem_u32(answer)) : "memory");
  x = (int)bx; y = (int)by;
  return got != 0;
}

// D(tmem) (+)= A(smem) * B(smem)^T and A(tmem) * B(smem), 16-bit operands, 32-bit sums. A whole warp comes here, and the lane
// with `leader` issues: a predicate instead of a branch lets the operands be computed in uniform registers, which is where the
// instruction takes them from. (A test of its own in front of each instruction undoes that, at 100 cycles an instruction: products
// of fewer channels or keys than a tile has run over the zeros there.)
__device__ __forceinline__ void umma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add)
{
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add ? 1 : 0), "r"(leader) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add)
{
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add ? 1 : 0), "r"(leader) : "memory");
}
__device__ __forceinline__ void umma_commit_by(uint32_t leader, uint64_t *bar)
{
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
               "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)), "r"(leader) : "memory");
}
__device__ __forceinline__ uint32_t elect_one()
{
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
// Shared-memory descriptors, whose low word holds the address in 16-byte units: the rest is the same for every tile.
// Q and K: rows of 128 bytes, swizzled, groups of 8 rows 1024 bytes apart. V as it lies, keys x channels: the product's N
// (channels) is contiguous, blocks of 64 channels are a box apart (leading offset), groups of 8 keys 1024 bytes (stride offset).
constexpr uint32_t DESC_HIGH = (1024u >> 4) | 1u << 14 | 2u << 29, DESC_K_LOW = 1u << 16, DESC_V_LOW = (128u * 128u >> 4) << 16;
__device__ __forceinline__ uint64_t desc_of(uint32_t low)
{
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low), "r"(DESC_HIGH));
  return d;
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
template <> struct Kind<__half> { static constexpr bool BF16 = false; static constexpr unsigned EXP = 0x7c00u; static constexpr float UNDER = 5.f; };
template <> struct Kind<__nv_bfloat16> { static constexpr bool BF16 = true; static constexpr unsigned EXP = 0x7f80u; static constexpr float UNDER = 0.f; };

__device__ __forceinline__ void make_work(Work &w, int q0, int lq, int k0, int lk, int pair, int kvh, const PromptProblem &p)
{
  w.q0 = q0; w.k0 = k0; w.lk = lk; w.kvh = kvh;
  w.lo = 0x7fffffff; w.hi = 0;
  for (int x = 0; x < 2; x++) {
    const int n = p.units * pair + x, rt = p.by_group.div(n);
    Unit u;
    u.row0 = rt * BQ; u.head = kvh * p.group + n - rt * p.group;
    u.rows = x < p.units ? min(max(lq - u.row0, 0), BQ) : 0;
    u.pos = u.row0 + lk - lq;
    const int keys = u.rows == 0 ? 0 : (p.causal ? min(lk, max(u.pos + u.rows, 0)) : lk);       // it sees none from here on
    const int from = p.window > 0 ? max(0, u.pos - p.window + 1) : 0;
    u.lo = from / BK; u.hi = (keys + BK - 1) / BK;
    if (from >= keys) u.lo = u.hi = 0;
    else { w.lo = min(w.lo, u.lo); w.hi = max(w.hi, u.hi); }
    w.u[x] = u;
  }
  w.lo = min(w.lo, w.hi);
}
__device__ __forceinline__ bool sees(const Unit &u, int j) { return j >= u.lo && j < u.hi; }
// whether some row of the unit does not see some key of tile j
__device__ __forceinline__ bool masked(const Unit &u, int j, int lk, const PromptProblem &p)
{
  const int k = j * BK, end = p.causal ? min(lk, u.pos + 1) : lk;
  return k + BK > end || (p.window > 0 && k < u.pos + u.rows - p.window);
}
__device__ __forceinline__ bool guarded(const Work &w, int j, const PromptProblem &p)
{
  return (sees(w.u[0], j) && masked(w.u[0], j, w.lk, p)) || (sees(w.u[1], j) && masked(w.u[1], j, w.lk, p));
}

// Finds pair number x of the units of all sequences: the longest first (`merged`), or in the sequences' order, where the search goes
// on where the last one stopped, `before` pairs lying ahead of sequence s0. A whole warp; false where there are not so many pairs.
__device__ __forceinline__ bool find_item(const PromptProblem &p, int x, int y, int lane, int &s0, int &before, Item &it)
{
  const bool merged = p.merged;
  for (; s0 < p.seqs; s0 += 256) {              // eight sequences a lane
    int at[9], at_k[9], count[8], sum = 0;
    const int b0 = s0 + lane * 8;
#pragma unroll
    for (int k = 0; k < 9; k++) {
      at[k] = b0 + k <= p.seqs ? min(max(__ldg(p.cu_q + b0 + k), 0), p.nq) : 0;
      at_k[k] = b0 + k <= p.seqs ? min(max(__ldg(p.cu_k + b0 + k), 0), p.nk) : 0;
    }
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const int tiles = b0 + k < p.seqs ? (max(at[k + 1] - at[k], 0) + BQ - 1) / BQ : 0;
      count[k] = (int)(((int64_t)tiles * p.group + p.units - 1) >> (p.units - 1));
      sum += count[k];
    }
    // merged: pair v of each sequence before pair v - 1 of any: as many pairs lie ahead of those numbered v as there are beyond
    // v in all sequences together.
    int v = 0;
    if (merged) {
      if ((unsigned)x >= __reduce_add_sync(0xffffffffu, (unsigned)sum)) return false;
      int most = 0;
#pragma unroll
      for (int k = 0; k < 8; k++) most = max(most, count[k]);
      int hi = __reduce_max_sync(0xffffffffu, most);
      unsigned ahead = 0;
      while (hi - v > 1) {               // the largest v with x < pairs numbered v and beyond
        const int mid = (v + hi) >> 1;
        unsigned n = 0;
#pragma unroll
        for (int k = 0; k < 8; k++) n += max(count[k] - mid, 0);
        n = __reduce_add_sync(0xffffffffu, n);
        if ((unsigned)x < n) v = mid;
        else { hi = mid; ahead = n; }
      }
      x -= (int)ahead; sum = 0;
#pragma unroll
      for (int k = 0; k < 8; k++) sum += count[k] > v;
    }
    int incl = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int n = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += n;
    }
    int off = before + incl - sum, q0 = 0, lq = 0, k0 = 0, lk = 0, pair = -1;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const int n = merged ? count[k] > v : count[k];
      if (x >= off && x < off + n) {
        // the last rows of a causal sequence see the most keys: they begin first
        q0 = at[k]; lq = at[k + 1] - at[k]; k0 = at_k[k]; lk = max(at_k[k + 1] - at_k[k], 0); pair = merged ? v : count[k] - 1 - (x - off);
      }
      off += n;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, pair >= 0);
    if (hit) {
      if (lane == __ffs(hit) - 1) make_work(it.w, q0, lq, k0, lk, pair, y, p);
      __syncwarp();
      return true;
    }
    if (merged) return false;
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

// Warps 10 and 11: the guards of the V tiles; warp 10 also fetches the items.
template <typename T, int DP>
__device__ __forceinline__ void guard_warp(Control &ct, char *smem, const PromptProblem &p, bool fetches, int id)
{
  using SH = Shape<DP>;
  constexpr int ST = SH::STAGES;
  constexpr unsigned E = Kind<T>::EXP;
  volatile int *abort_flag = &ct.abort_flag;
  const int lane = id & 31;
  int s0 = 0, before = 0, row = blockIdx.y, asked = 0;
  bool ok = true, pending = false;
  // publishes item number i
  auto publish = [&](int i) {
    ok = __all_sync(0xffffffffu, mbar_wait(&ct.item_empty[i % ITEMS], ((i / ITEMS) & 1) ^ 1, abort_flag, p.status, ST_GUARD));
    Item &it = ct.item[i % ITEMS];
    bool own = i == 0, found = false;
    while (ok) {
      int x = blockIdx.x, y = blockIdx.y;
      bool got = true;
      if (!own) {
        ok = __all_sync(0xffffffffu, mbar_wait(&ct.next, (asked - 1) & 1, abort_flag, p.status, ST_GUARD));
        if (!ok) break;
        pending = false;
        got = block_of(&ct.answer, x, y);
        fence_proxy_async();                   // the next answer comes behind these reads
        __syncwarp();
      }
      own = false;
      if (!got) break;                         // nothing is left, and nothing may be asked for again
      if (lane == 0) ask_for_block(&ct.answer, &ct.next);
      asked++; pending = true;
      if (y != row || x < before) { row = y; s0 = 0; before = 0; }
      if ((found = find_item(p, x, y, lane, s0, before, it))) break;
      // a block beyond the last pair: the grid is made for the most there can be
    }
    if (lane == 0) {
      it.end = !found; it.dirty = 0;
      mbar_arrive(&ct.item_full[i % ITEMS]);
    }
    __syncwarp();
  };
  if (fetches) publish(0);
  int e = 1;                                   // the ring's number of the next V tile
  for (int i = 0; ok; i++) {
    ok = __all_sync(0xffffffffu, mbar_wait(&ct.item_full[i % ITEMS], (i / ITEMS) & 1, abort_flag, p.status, ST_GUARD));
    if (!ok || ct.item[i % ITEMS].end) break;
    const Work &w = ct.item[i % ITEMS].w;
    if (fetches) publish(i + 1);
    const int lo = w.lo, hi = w.hi;
    for (int j = lo; j < hi && ok; j++, e += 2) {
      const int st = e % ST;
      ok = __all_sync(0xffffffffu, mbar_wait(&ct.kv_full[st], (e / ST) & 1, abort_flag, p.status, ST_GUARD));
      if (!ok) break;
      if (guarded(w, j, p)) {
        const int rows = w.lk - j * BK;
        bool odd = false;
        for (int k = id; k < SH::TILE / 16; k += GUARD_THREADS) {
          uint4 *at = reinterpret_cast<uint4 *>(smem + (2 + st) * SH::TILE) + k;
          if (((k >> 3) & 127) >= rows) { *at = make_uint4(0, 0, 0, 0); continue; }
          const uint4 v = *at;
          // the exponent's bits all set: adding one at their lowest place carries into the sign's
          auto bad = [](unsigned v) { return ((v & (E * 0x10001u)) + (E & (~E + 1u)) * 0x10001u) & 0x80008000u; };
          const unsigned a = bad(v.x), b = bad(v.y), c = bad(v.z), d = bad(v.w);
          if (a | b | c | d) {
            auto keep = [](unsigned v, unsigned b) { return v & ~((b >> 15) * 0xffffu); };
            *at = make_uint4(keep(v.x, a), keep(v.y, b), keep(v.z, c), keep(v.w, d));
            odd = true;
          }
        }
        if (odd) *reinterpret_cast<volatile int *>(&ct.item[i % ITEMS].dirty) = 1;
        fence_proxy_async();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ct.clean[st >> 1]);
    }
    if (lane == 0) mbar_arrive(&ct.item_empty[i % ITEMS]);
  }
  if (pending) {          // given up with a request under way: its answer must land first
    volatile int never = 0;
    mbar_wait(&ct.next, (asked - 1) & 1, &never, nullptr, 0);
  }
}

__device__ __noinline__ bool wait_long(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int *status, int code)
{
  return mbar_wait(bar, parity, abort_flag, status, code);
}

// Warp 9: issues the MMAs. The whole warp walks through the tiles, so that what the instructions take from uniform
// registers is computed there; one lane issues and commits.
template <typename T, int DP>
__device__ __forceinline__ void mma_warp(Control &ct, uint32_t base, uint32_t tmem_, const PromptProblem &p)
{
  using SH = Shape<DP>;
  constexpr int ST = SH::STAGES;
  volatile int *abort_flag = &ct.abort_flag;
  const uint32_t leader = elect_one();
  // a wait that fails is looked at once a tile only: until then products of stale tiles do no harm, their results are void
  bool ok = true;
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (!mbar_try_wait(bar, parity)) ok = wait_long(bar, parity, abort_flag, p.status, ST_MMA) && ok;
  };
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_, 0);
  const uint32_t q_low = __shfl_sync(0xffffffffu, ((base & 0x3ffffu) >> 4) | DESC_K_LOW, 0);
  const uint32_t k_low = __shfl_sync(0xffffffffu, (((base + 2 * SH::TILE) & 0x3ffffu) >> 4) | DESC_K_LOW, 0);
  const uint32_t v_low = __shfl_sync(0xffffffffu, (((base + 2 * SH::TILE) & 0x3ffffu) >> 4) | DESC_V_LOW, 0);
  const uint32_t id_s = idesc16(Kind<T>::BF16, false, BK), id_o = idesc16(Kind<T>::BF16, true, (p.dim + 15) / 16 * 16);
  int i = -1, np[2] = {0, 0}, nq[2] = {0, 0}, ns[2] = {0, 0}, e = 0;        // e: the ring's number of the current key tile
  struct Range { int lo, hi, ulo[2], uhi[2]; } cur, nxt;      // key tiles of an item and of its units
  // Looks at the next item. TILES: it has key tiles; NONE: it needs nothing here; END: there is none, or an error (ok).
  enum Next { END, NONE, TILES };
  auto next_item = [&](Range &r) {
    i++;
    wait(&ct.item_full[i % ITEMS], (i / ITEMS) & 1);
    if (__any_sync(0xffffffffu, !ok) || __any_sync(0xffffffffu, ct.item[i % ITEMS].end)) return END;
    const Work &w = ct.item[i % ITEMS].w;
    r.lo = __shfl_sync(0xffffffffu, w.lo, 0); r.hi = __shfl_sync(0xffffffffu, w.hi, 0);
#pragma unroll
    for (int x = 0; x < 2; x++) {
      r.ulo[x] = __shfl_sync(0xffffffffu, w.u[x].lo, 0); r.uhi[x] = __shfl_sync(0xffffffffu, w.u[x].hi, 0);
    }
    __syncwarp();
    if (leader) mbar_arrive(&ct.item_empty[i % ITEMS]);
    return r.lo < r.hi ? TILES : NONE;
  };
  auto wait_kv = [&](int k) { wait(&ct.kv_full[k % ST], (k / ST) & 1); };
  // S of unit x with tile j, K being number k of the ring, which has landed
  auto issue_s = [&](int x, int lo, int hi, int j, int k) {
    if (j == lo) {
      wait(&ct.q_full[x], nq[x] & 1);
      nq[x]++;
      tc_fence_after();
    }
    if (SH::APART && ns[x] > 0) {              // the softmax has the last S in registers
      wait(&ct.s_free[x], (ns[x] - 1) & 1);
      tc_fence_after();
    }
    ns[x]++;
    const uint32_t a = q_low + x * (SH::TILE >> 4), b = k_low + (k % ST) * (SH::TILE >> 4);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ks++) {
      const uint32_t off = ((ks >> 2) * SH::BOX + (ks & 3) * 32) >> 4;
      umma_ss(leader, tmem + x * 128, desc_of(a + off), desc_of(b + off), id_s, ks > 0);
    }
    umma_commit_by(leader, &ct.s_full[x]);
    if (j == hi - 1) umma_commit_by(leader, &ct.q_empty[x]);
  };
  Next next = next_item(cur);
  while (true) {
    // the first S of an item behind which no product is left to issue
    while (next == NONE) next = next_item(cur);
    if (next == END) break;
    int j = cur.lo;
    wait_kv(e);
    if (__any_sync(0xffffffffu, !ok)) break;
    tc_fence_after();
#pragma unroll
    for (int x = 0; x < 2; x++)
      if (j >= cur.ulo[x] && j < cur.uhi[x]) issue_s(x, cur.ulo[x], cur.uhi[x], j, e);
    umma_commit_by(leader, &ct.kv_empty[e % ST]);
    bool more = true;                          // S of a next tile has been issued, too
    while (more) {
      // The tile after this one, of this item or the next. Where the next item has none, this tile's P V goes out before a further
      // item is looked at: items come as earlier ones are done (ITEMS at a time), and this one is not before its last P V.
      const bool same = j + 1 < cur.hi;
      int jn = j + 1;
      if (!same) {
        next = next_item(nxt);
        more = next == TILES;
        jn = nxt.lo;
      }
      wait_kv(e + 1);
      wait(&ct.clean[((e + 1) % ST) >> 1], ((e + 1) / ST) & 1);
      if (more) wait_kv(e + 2);
      if (__any_sync(0xffffffffu, !ok)) { next = END; break; }
      const uint32_t b = v_low + ((e + 1) % ST) * (SH::TILE >> 4);
      auto next_s = [&](int x) {
        const int lo_n = same ? cur.ulo[x] : nxt.ulo[x], hi_n = same ? cur.uhi[x] : nxt.uhi[x];
        if (more && jn >= lo_n && jn < hi_n) issue_s(x, lo_n, hi_n, jn, e + 2);
      };
      if (SH::APART) {
#pragma unroll
        for (int x = 0; x < 2; x++) next_s(x);
      }
#pragma unroll
      for (int x = 0; x < 2; x++) {
        if (j >= cur.ulo[x] && j < cur.uhi[x]) {
          const bool begun = j > cur.ulo[x], last = j == cur.uhi[x] - 1;
          const uint32_t o = tmem + SH::O_AT + x * DP, w = tmem + SH::P_AT + x * SH::P_STEP;
          if (!SH::APART) {
            wait(&ct.p_half[x], np[x] & 1);
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < 4; kk++) umma_ts(leader, o, w + kk * 8, desc_of(b + kk * (2048 >> 4)), id_o, begun || kk > 0);
            umma_commit_by(leader, &ct.pv_done[x]);         // of the first half
          }
          wait(&ct.p_full[x], np[x] & 1);
          np[x]++;
          tc_fence_after();
#pragma unroll
          for (int kk = SH::APART ? 0 : 4; kk < 8; kk++) umma_ts(leader, o, w + kk * 8, desc_of(b + kk * (2048 >> 4)), id_o, begun || kk > 0);
          if (SH::APART) umma_commit_by(leader, &ct.pv_done[x]);
          if (last) umma_commit_by(leader, &ct.o_full[x]);
        }
        if (!SH::APART) next_s(x);
      }
      umma_commit_by(leader, &ct.kv_empty[(e + 1) % ST]);
      if (more) umma_commit_by(leader, &ct.kv_empty[(e + 2) % ST]);
      e += 2;
      j = jn;
      if (!same) cur = nxt;
    }
  }
  // the MMAs issued so far end before TMEM is given back
  volatile int never = 0;
  umma_commit_by(leader, &ct.drain);
  mbar_wait(&ct.drain, 0, &never, p.status, ST_MMA);
}

// two values in a register pair, one instruction for both
__device__ __forceinline__ uint64_t pair2(float a, float b)
{
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 both(uint64_t v)
{
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// mbar_wait of a whole warp, which goes on or gives up as one. The vote is the loop's own condition, so that the lanes never part: 24 packed
// prompts 209.6 us, 215 with lanes that wait each by themselves and vote then.
__device__ __forceinline__ bool wait_together(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int *status, int code)
{
  unsigned long long t0 = 0;
  for (unsigned spin = 1; !__all_sync(0xffffffffu, mbar_try_wait(bar, parity)); spin++) {
    if ((spin & 255u) == 0) {
      const unsigned long long now = global_ns();
      if (t0 == 0) t0 = now;
      const bool late = now - t0 > WAIT_LIMIT_NS;
      if (late) {
        *abort_flag = 1;
        if (status) atomicOr(status, code);
      }
      if (__any_sync(0xffffffffu, late || *abort_flag)) return false;
    }
  }
  return true;
}

// Warps 0 to 7: the softmax of a unit, a row a thread.
template <typename T, int DP>
__device__ __forceinline__ void softmax_warps(Control &ct, uint32_t staging, uint32_t tmem, const PromptProblem &p)
{
  using SH = Shape<DP>;
  volatile int *abort_flag = &ct.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, x = warp >> 2, r = threadIdx.x & 127;
  const uint32_t rowbase = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  const uint32_t t_s = rowbase + x * 128, t_o = rowbase + SH::O_AT + x * DP, t_p = rowbase + SH::P_AT + x * SH::P_STEP;
  const int groups = (p.dim + 15) / 16;
  uint32_t done = 0, o_phase = 0;              // tiles of this unit; item ends
  // A whole warp goes on or gives up, since loads and stores of TMEM want all its lanes.
  auto waited = [&](uint64_t *bar, uint32_t parity, int code) { return wait_together(bar, parity, abort_flag, p.status, code); };
  bool ok = true;
  for (int i = 0; ok; i++) {
    if (!(ok = waited(&ct.item_full[i % ITEMS], (i / ITEMS) & 1, ST_SOFTMAX))) break;
    const Item &it = ct.item[i % ITEMS];
    if (it.end) break;
    const Unit w = it.w.u[x];
    const int lk = it.w.lk;
    const int pos = w.pos + r;
    const int last = p.causal ? min(lk - 1, pos) : lk - 1, first = p.window > 0 ? pos - p.window + 1 : 0;
    // every row sees every key of the tiles whole_lo .. whole_hi - 1
    const int whole_hi = (p.causal ? min(lk, max(w.pos + 1, 0)) : lk) / BK, whole_lo = p.window > 0 ? (max(w.pos + w.rows - p.window, 0) + BK - 1) / BK : 0;
    float m = NOTHING, l = 0.f;
    bool far = false;                          // some row's reference is beyond 2^24
    for (int j = w.lo; j < w.hi; j++, done++) {
      if (!(ok = waited(&ct.s_full[x], done & 1, ST_SOFTMAX))) break;
      tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int k = 0; k < 4; k++) tmem_ld_32(t_s + k * 32, s[k]);
      tmem_wait_ld();
      if (SH::APART) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ct.s_free[x]);
      }
      if (j >= whole_hi || j < whole_lo) {
        const int a = first - j * BK, b = last - j * BK;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          // bit c: whether the row sees key 32 k + c of the tile. One test of a bit a score; two comparisons took the packed
          // prompts above from 215 to 230 us
          const int from = a - k * 32, to = b - k * 32;
          const unsigned seen = (from <= 0 ? 0xffffffffu : (from < 32 ? 0xffffffffu << from : 0u)) & (to >= 31 ? 0xffffffffu : (to >= 0 ? 0xffffffffu >> (31 - to) : 0u));
#pragma unroll
          for (int c = 0; c < 32; c++)
            if (!(seen & (1u << c))) s[k][c] = 0xff800000u;
        }
      }
      float scale = p.scale_log2;
      // A new reference: the maximum so far. O is rescaled where it holds something (`has`); its products have ended.
      auto raise = [&](bool has) {
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 32; c += 2)
#pragma unroll
          for (int k = 0; k < 4; k++) top[k] = max3(top[k], __uint_as_float(s[k][c]), __uint_as_float(s[k][c + 1]));
        const float most = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * scale;
        if (!(most <= 3.402823466e38f)) l = __int_as_float(0x7fffffff);        // a NaN or an infinity among the scores
        const float to = fmaxf(m, most - Kind<T>::UNDER), f = ex2(m - to);
        m = to;
        far = __any_sync(0xffffffffu, fabsf(m) > 16777216.f && m > NOTHING);
        l *= f;
        if (has) {
          for (int c = 0; c < groups; c++) {
            uint32_t o[16];
            tmem_ld_16(t_o + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            tmem_st_16(t_o + c * 16, o);
          }
        }
      };
      // Scores are scaled within the subtraction of the reference, which is rounded once. Against a reference that is itself a rounded
      // product, beyond 2^24 that leaves whole units of its last place, of either sign, for weights to be 2 to the power of.
      // There (`far`) the scores are scaled and rounded first, as the reference was. At 64 channels a scale that changes costs
      // registers (215 us instead of 207 for the packed prompts above): the differences, in units of the score, take the scores' place;
      // at 128 channels that and its second maximum take longer (300 tokens 11.7 us, so 11.3).
      auto scale_first = [&] {
        if (SH::APART) {
          const float back = 1.f / p.scale_log2;
#pragma unroll
          for (int k = 0; k < 4; k++)
#pragma unroll
            for (int c = 0; c < 32; c++) s[k][c] = __float_as_uint((__fmul_rn(__uint_as_float(s[k][c]), p.scale_log2) - m) * back);
        } else {
#pragma unroll
          for (int k = 0; k < 4; k++)
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              const float2 v = both(mul2(pair2(__uint_as_float(s[k][c]), __uint_as_float(s[k][c + 1])), pair2(scale, scale)));
              s[k][c] = __float_as_uint(v.x); s[k][c + 1] = __float_as_uint(v.y);
            }
          scale = 1.f;
        }
      };
      // the weights of 32 keys, as the second product wants them, and their sum
      auto weights = [&](int k, uint64_t off2) {
        uint64_t sum = 0;
        const uint64_t scale2 = pair2(scale, scale);
        uint32_t w16[16];
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          const uint64_t a = fma2(pair2(__uint_as_float(s[k][c]), __uint_as_float(s[k][c + 1])), scale2, off2);
          const float2 e = make_float2(ex2(both(a).x), ex2(both(a).y));
          sum = add2(sum, pair2(e.x, e.y));
          w16[c / 2] = pack2<T>(e.x, e.y);       // off by 2^-8 (bf16) or 2^-11 (fp16) of each weight at most; their sum is taken unrounded
        }
        tmem_st_16(t_p + k * 16, w16);
        return sum;
      };
      auto hand_over = [&](uint64_t *bar) {
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
      };
      // With the reference as it is; with a new one where there is none yet, or where the weights' sum shows that one of them is
      // beyond 2^15 (or no number). In between, the scores' maximum is not looked for: that took a fifth of the time.
      if (SH::APART) {
        if (!(ok = waited(&ct.pv_done[x], (done - 1) & 1, ST_SOFTMAX))) break;      // of the tile before; there is none to wait for before the first
        tc_fence_after();
        bool raised = false, need = j == w.lo || far;
        while (true) {
          if (need) { raise(j > w.lo); raised = true; if (far) scale_first(); }
          const float off = far ? 0.f : -m;
          const uint64_t off2 = pair2(off, off);
          uint64_t sum[4];
#pragma unroll
          for (int k = 0; k < 4; k++) sum[k] = weights(k, off2);
          const float2 v = both(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
          if (raised || !__any_sync(0xffffffffu, !(v.x + v.y < 32768.f))) { l += v.x + v.y; break; }
          need = true;
        }
        hand_over(&ct.p_full[x]);
      } else {
        bool raised = j == w.lo;
        if (raised) raise(false);
        if (far) scale_first();
#pragma unroll
        for (int h = 0; h < 2; h++) {
          while (true) {
            const uint64_t off2 = pair2(-m, -m);
            const uint64_t a = weights(2 * h, off2), b = weights(2 * h + 1, off2);
            const float2 v = both(add2(a, b));
            if (raised || !__any_sync(0xffffffffu, !(v.x + v.y < 32768.f))) { l += v.x + v.y; break; }
            raised = true;
            // the second half: the first half's product must have ended before O is rescaled
            if (h == 1) {
              if (!(ok = waited(&ct.pv_done[x], done & 1, ST_SOFTMAX))) break;
              tc_fence_after();
            }
            raise(h == 1 || j > w.lo);
            if (far) scale_first();
          }
          if (!ok) break;
          hand_over(h == 0 ? &ct.p_half[x] : &ct.p_full[x]);
        }
        if (!ok) break;
      }
    }
    if (!ok) break;
    // ---- the rows ----
    const bool any = w.hi > w.lo;
    if (any) {
      if (!(ok = waited(&ct.o_full[x], o_phase, ST_EPI))) break;
      o_phase ^= 1;
      tc_fence_after();
    }
    const bool live = r < w.rows;
    const int64_t row = it.w.q0 + w.row0 + r;
    const float inv = l == 0.f ? 0.f : 1.f / l;         // a row that sees nothing is zero: its O is, the guards having been over V
    char *dst = p.out + row * p.out_row + (int64_t)w.head * p.out_head;
    const bool dirty = any && *reinterpret_cast<const volatile int *>(&it.dirty);
    // 16-bit rows go through shared memory, 64 channels at a time, and leave as whole rows: stored by their own threads, each
    // instruction would touch 32 rows (300 tokens of 32 heads: 4900 of 24000 cycles)
    const uint32_t stage = staging + warp * SH::STAGING;
    // eight lanes write 64 channels of a row: rows 4 k + lane / 8 of the warp's 32
    const int chunk = lane & 7;
    auto store = [&](int c) {
      const int channel = (c & ~3) * 16 + chunk * 8;
      char *to = p.out + ((int64_t)it.w.q0 + w.row0 + (warp & 3) * 32) * p.out_row + (int64_t)w.head * p.out_head + channel * 2;
      __syncwarp();
      uint4 v[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int n = k * 4 + (lane >> 3);
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[k].x), "=r"(v[k].y), "=r"(v[k].z), "=r"(v[k].w) : "r"(stage + n * 128 + ((chunk ^ (n & 7)) << 4)) : "memory");
      }
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int n = k * 4 + (lane >> 3);
        if ((warp & 3) * 32 + n < w.rows && channel < p.dim) *reinterpret_cast<uint4 *>(to + n * p.out_row) = v[k];
      }
      __syncwarp();
    };
    // By far the most items, without the tests below: packed prompts 209 us with it, 215 without. (Two or four groups at a time cost
    // the main loop its registers: 222, 272.)
    const bool plain = any && !dirty && p.out_type != PULPNN_TYPE_U8;
#pragma unroll 1
    for (int c = 0; plain && c < groups; c++) {
      uint32_t o[16];
      tmem_ld_16(t_o + c * 16, o);
      tmem_wait_ld();
#pragma unroll
      for (int k = 0; k < 2; k++) {
        uint32_t w4[4];
#pragma unroll
        for (int e = 0; e < 4; e++) w4[e] = pack2<T>(__uint_as_float(o[8 * k + 2 * e]) * inv, __uint_as_float(o[8 * k + 2 * e + 1]) * inv);
        sts128(stage + lane * 128 + ((((c & 3) * 2 + k) ^ (lane & 7)) << 4), w4[0], w4[1], w4[2], w4[3]);
      }
      if ((c & 3) == 3 || c == groups - 1) store(c);
    }
    for (int c = plain ? groups : 0; c < groups; c++) {
      float y[16];
      if (any) {
        uint32_t o[16];
        tmem_ld_16(t_o + c * 16, o);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 16; k++) y[k] = __uint_as_float(o[k]) * inv;
      } else {
#pragma unroll
        for (int k = 0; k < 16; k++) y[k] = 0.f;
      }
      if (dirty && live) {      // the infinities and NaN that the guards took out of the tiles, where this row sees them
        const Work &all = it.w;
        for (int j = w.lo; j < w.hi; j++) {
          if (!guarded(all, j, p)) continue;
          for (int k = max(first, j * BK); k <= min(last, j * BK + BK - 1); k++) {
            const T *v = reinterpret_cast<const T *>(p.v + (int64_t)(all.k0 + k) * p.v_row + (int64_t)all.kvh * p.v_head) + c * 16;
#pragma unroll
            for (int n = 0; n < 16; n++)
              if (c * 16 + n < p.dim) {
                const float z = (float)v[n];
                if (!(fabsf(z) <= 3.402823466e38f)) y[n] += z;
              }
          }
        }
      }
      __syncwarp();             // the rows' keys differ; the next group's load wants the whole warp
      if (p.out_type == PULPNN_TYPE_U8) {
        if (live) {
#pragma unroll
          for (int k = 0; k < 16; k += 4)
            if (c * 16 + k < p.dim) {
              const float z[4] = {y[k], y[k + 1], y[k + 2], y[k + 3]};
              store4(dst, c * 16 + k, p.out_type, z, p.out_inv_step, p.out_zero);
            }
        }
        continue;
      }
#pragma unroll
      for (int k = 0; k < 2; k++)
        sts128(stage + lane * 128 + ((((c & 3) * 2 + k) ^ (lane & 7)) << 4), pack2<T>(y[8 * k], y[8 * k + 1]), pack2<T>(y[8 * k + 2], y[8 * k + 3]),
               pack2<T>(y[8 * k + 4], y[8 * k + 5]), pack2<T>(y[8 * k + 6], y[8 * k + 7]));
      if ((c & 3) == 3 || c == groups - 1) store(c);
    }
    if (live && p.lse) p.lse[row * p.hq + w.head] = (m + __log2f(l)) * 0.69314718055994530942f;      // log2 l: off by 2^-22 or 2 units in its last place
    tc_fence_before();          // O has been read: the next item's first P, behind this, lets it be written over
    __syncwarp();
    if (lane == 0) mbar_arrive(&ct.item_empty[i % ITEMS]);
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, 1)
attn_prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const PromptProblem p)
{
  using SH = Shape<DP>;
  constexpr int ST = SH::STAGES;
  extern __shared__ char raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  char *smem = raw + (base - smem_u32(raw));
  Control &ct = *reinterpret_cast<Control *>(smem + (2 + ST) * SH::TILE);
  static_assert(sizeof(Control) <= 1024, "control block");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int *abort_flag = &ct.abort_flag;

  if (threadIdx.x == 0) {
    ct.abort_flag = 0;
    for (int x = 0; x < 2; x++) {
      mbar_init(&ct.q_full[x], 1); mbar_init(&ct.q_empty[x], 1); mbar_init(&ct.s_full[x], 1); mbar_init(&ct.o_full[x], 1);
      mbar_init(&ct.s_free[x], 4); mbar_init(&ct.p_half[x], 4); mbar_init(&ct.p_full[x], 4); mbar_init(&ct.pv_done[x], 1);
    }
    for (int s = 0; s < ST; s++) { mbar_init(&ct.kv_full[s], 1); mbar_init(&ct.kv_empty[s], 1); }
    for (int s = 0; s < ST / 2; s++) mbar_init(&ct.clean[s], 2);
    for (int s = 0; s < ITEMS; s++) { mbar_init(&ct.item_full[s], 1); mbar_init(&ct.item_empty[s], 12); }      // every warp is done with an item
    mbar_init(&ct.next, 1); mbar_init(&ct.drain, 1);
    mbar_fence_init();
  }
  if (warp == WARP_MMA) tmem_alloc(&ct.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ct.tmem;
  pdl_wait();

  // item number i; false where an error ends the kernel
  auto wait_item = [&](int i, int code) { return mbar_wait(&ct.item_full[i % ITEMS], (i / ITEMS) & 1, abort_flag, p.status, code); };

  if (warp >= WARP_LOAD) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == WARP_LOAD) {
      if (lane == 0) {
        int e = 0, nq[2] = {0, 0};
        bool ok = true;
        for (int i = 0; ok; i++) {
          if (!(ok = wait_item(i, ST_LOAD)) || ct.item[i % ITEMS].end) break;
          const Work &w = ct.item[i % ITEMS].w;
          const int hi = w.hi, kvh = w.kvh, k0 = w.k0;
#pragma unroll
          for (int x = 0; x < 2; x++) {
            if (!ok || w.u[x].hi <= w.u[x].lo) continue;
            if (nq[x] > 0 && !(ok = mbar_wait(&ct.q_empty[x], (nq[x] - 1) & 1, abort_flag, p.status, ST_LOAD))) continue;
            mbar_arrive_expect_tx(&ct.q_full[x], SH::TILE);
            for (int b = 0; b < SH::BOXES; b++)
              tma_load_3d(smem + x * SH::TILE + b * SH::BOX, &map_q, &ct.q_full[x], b * 64, w.u[x].head, w.q0 + w.u[x].row0);
            nq[x]++;
          }
          for (int j2 = 2 * w.lo; j2 < 2 * hi && ok; j2++) {
            const int st = e % ST;
            if (!(ok = mbar_wait(&ct.kv_empty[st], ((e / ST) & 1) ^ 1, abort_flag, p.status, ST_LOAD))) break;
            mbar_arrive_expect_tx(&ct.kv_full[st], SH::TILE);
            for (int b = 0; b < SH::BOXES; b++)
              tma_load_3d(smem + (2 + st) * SH::TILE + b * SH::BOX, e & 1 ? &map_v : &map_k, &ct.kv_full[st], b * 64, kvh, k0 + (j2 >> 1) * BK);
            e++;
          }
          mbar_arrive(&ct.item_empty[i % ITEMS]);
        }
        if (!ok) {        // given up: the copies in flight must land before the CTA's shared memory is given away
          volatile int never = 0;
#pragma unroll
          for (int x = 0; x < 2; x++)
            if (nq[x] > 0) mbar_wait(&ct.q_full[x], (nq[x] - 1) & 1, &never, nullptr, 0);
          for (int k = max(0, e - ST); k < e; k++) mbar_wait(&ct.kv_full[k % ST], (k / ST) & 1, &never, nullptr, 0);
        }
      }
    } else if (warp == WARP_MMA) {
      mma_warp<T, DP>(ct, base, tmem, p);
    } else {
      guard_warp<T, DP>(ct, smem, p, warp == WARP_GUARD, threadIdx.x - WARP_GUARD * 32);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    softmax_warps<T, DP>(ct, base + (2 + ST) * SH::TILE + 1024, tmem, p);
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
  // The grid is made for the most items that so many sequences may have. What empty ones leave of it is taken over block by block, at 0.33 us a
  // block and SM, and sequences are looked through 256 at a time, while the other warps wait: 0.4 s within these bounds; the waits end after 1 s.
  ATTN_REQUIRE(a->n_seqs <= 1 << 24 && (int64_t)a->n_seqs * a->n_heads <= 1 << 26, PULPNN_ERR_UNSUPPORTED, "%s: %d sequences of %d heads", who, a->n_seqs, a->n_heads);
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
  p.nq = a->n_q_rows; p.nk = a->n_k_rows; p.seqs = a->n_seqs; p.hq = a->n_heads; p.group = a->n_heads / a->n_kv_heads; p.by_group.set((unsigned)p.group); p.dim = a->head_dim;
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
  // at most so many units: a sequence's rows fill all its tiles but one; and items, of which a sequence's last may be half empty
  const int64_t units = ((int64_t)a->n_q_rows / BQ + a->n_seqs) * p.group;
  // one unit an item where that still fits the GPU at once: 300 tokens of 32 heads took 12.9 us, 13.9 in pairs
  p.units = units * a->n_kv_heads <= c.sm_count ? 1 : 2;
  const int64_t pairs = p.units == 1 ? units : (units + a->n_seqs + 1) / 2;
  // Longest first, so that no SM begins a long item last: 24 packed prompts of 1 to 2048 tokens 230 us, 247 in the sequences' order; 250
  // of 300 tokens 549 and 633. A warp looks through up to 256 sequences at once, which takes longer than to go on from the last one
  // and shows where an SM has few items: two prompts of 500 tokens 16.7 us, 14.4 in order.
  p.merged = a->n_seqs > 1 && a->n_seqs <= 256 && pairs * a->n_kv_heads >= 12 * (int64_t)c.sm_count;
  ATTN_REQUIRE(pairs <= 0x3fffffff, PULPNN_ERR_UNSUPPORTED, "%s: %d rows in %d sequences", who, a->n_q_rows, a->n_seqs);
  const dim3 grid((unsigned)pairs, (unsigned)a->n_kv_heads);
  const bool f16 = a->type == PULPNN_TYPE_F16, narrow = a->head_dim <= 64;
  const bool ok = f16 ? (narrow ? prompt_go<__half, 64>(c, mq, mk, mv, p, grid) : prompt_go<__half, 128>(c, mq, mk, mv, p, grid))
                      : (narrow ? prompt_go<__nv_bfloat16, 64>(c, mq, mk, mv, p, grid) : prompt_go<__nv_bfloat16, 128>(c, mq, mk, mv, p, grid));
  return ok ? PULPNN_OK : c.err;
}
