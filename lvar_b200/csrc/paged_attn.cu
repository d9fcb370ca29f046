// Attention of a few new tokens per sequence over the paged key/value cache:
//   o[b,h,t,:] = sum_j softmax_j(scale q[b,h,t].K[b,h/G,j]) V[b,h/G,j,:],  j < len_b  (causal: j <= len_b - T + t).
//
// Bound by reading the cache (4 D bytes per cached row in bf16, 2 D + 2 in e4m3; 4 D flops per row and query row): the
// G = Hq / Hkv query heads of a key head and the T tokens are the rows of one tile, so that a cached row crosses HBM
// once for all of them.  Products are warp-level matrix instructions (m16n8k16) with the keys, and in the second product the
// elements of V, along their 16 rows and the query rows along their 8 columns: S^T = K Q^T, O^T = V^T P^T, P^T made from S^T
// by an 8 x 8 transposition in registers.  One query row so pays for 8; the tensor-memory instructions start at 64, and
// their accumulators would have to come back through tensor memory for every step of the running softmax.  With up to 8 rows
// the tensor pipe is 15 to 17 % busy and HBM bounds the kernel (24 x 16 heads x 10521 keys in bf16: 313 to 320 us,
// 6.5 TB/s); with 64 rows tensor pipe (58 %) and shared memory (65 %) do (16 x 8 heads x 8192 keys: 122 us, 0.67 of HBM).
//
// A CTA is four warps that compute and one that loads.  The loader follows the page table (one lane per box of 16 to 128
// rows that lie together in a page) and streams tiles of keys through a ring in shared memory with tensor-map copies,
// swizzled; the others wait for a tile and hand its place back, and meet only at an item's end.  Rows of a box behind the
// sequence's end are copied too: their scores are masked and their V rows made zeros.  With up to 16 rows the four warps
// take a quarter of a tile's keys each and have a reference, sum and accumulator of their own, joined once at the end of the
// piece; with more rows (up to 64 per CTA) two or four warps share the keys and differ in their rows.
// (16-byte copies by all threads: 98 us for 16 x 8 heads x 8192 keys in e4m3; with the loader 68; keys along the 16 rows 55;
// the loader's registers to the others 53.)
//
// Split over the cache's length: all items (sequence, key head, row tile) lie on one line that the CTAs (two or three per SM) share
// evenly, whatever the lengths are: they are read on the device.  An item that falls to several CTAs leaves at most two pieces
// per CTA in the workspace (unnormalised sums, maximum, sum), and a second kernel joins them in a fixed order.  Where items
// are short a CTA takes one item and there is no second kernel (see plan_of).
//
// e4m3 cache: K and V rows are widened to fp16 (exact), q is scaled by a power of two per row into fp16's range: exact for
// elements down to 2^-17 of the row's largest; smaller ones are off by up to 2^-25 of it (fp16's steps end at 2^-24).  K's row scale multiplies the score.  V's row scale 2^e joins the exponent
// of the weight, w = exp2(s + e - reference of (s + e)), so that the fp16 weights are always taken relative to the
// largest CONTRIBUTION; the row sum keeps a maximum of its own.
// Weights against an e4m3 cache are rounded to fp16 (scaled by 2^7, so that only weights 2^-21 of the largest or less are
// subnormal).  Against a bf16 cache up to 16 rows take them as the sum of two bf16 numbers, 2^-17 of them off: rounded once
// they add as much again to the error of the output's own rounding, and next to HBM the second product and its look for
// elements of V that are not finite cost at most 1 % (24 x 16 heads x 10521 keys 311 us either way).  With more rows the
// matrix instructions count, and weights are rounded to bf16, 2^-8 of them off (16 x 8 heads x 8192 keys, one product / two:
// 32 rows 100 / 110 us, 48 rows 122 / 152, 64 rows 124 / 155; 16 x 4 heads x 35 rows x 4121 keys 31.7 / 35.9, error of the
// output 2.2e-3 / 1.7e-3 of its norm).  Sums, maxima and accumulators are fp32.
#include <math.h>

#include "paged.cuh"
#include "ptx.cuh"

namespace lvar {

namespace {

constexpr int kThreads = 128;     // threads that compute: a warpgroup
constexpr int kAllThreads = 256;  // and one whose first warp loads; its registers go to the first
constexpr int kSlotsPerCta = 2;
constexpr float kUp = 7.f;  // fp16 weights are scaled by 2^7; with 2^8 above the reference they end at 2^15

struct PagedAttnParams {
  PagedView c;
  const int32_t* lens;
  const __nv_bfloat16* q;
  int64_t q_sb, q_sh, q_sl;
  __nv_bfloat16* o;
  int64_t o_sb, o_sh, o_sl;
  float* M;  // [B, Hq, T] or null
  float* L;
  float* part;  // workspace of the split form: the CTAs' pieces,
  int4* heads;  // and what begins in a CTA's range and goes on behind it: sequence, head and row tile, pieces (0: none), slot
  int32_t* status;
  int B, Hkv, G, T, R;  // R = T * G rows per (sequence, key head)
  int RT;               // row tiles
  int causal, max_len;
  int split;            // 0: CTA x takes item x
  float scale_log2;
  int box_log2;         // rows per copy: 16 to 128
  uint64_t wait_limit_ns;
};

// An untiled copy of a multiple of 16 bytes between 16-byte aligned places.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory"); }
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four e4m3 bytes to two pairs of fp16 (exact); the lowest byte goes to the low half of `lo`.
__device__ __forceinline__ void widen4(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}"
      : "=r"(lo), "=r"(hi) : "r"(four));
}
// Transposes an 8 x 8 matrix of 16-bit elements held as an accumulator's rows.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// The larger magnitude of either half's two bf16, or NaN (with a sign that means nothing).
__device__ __forceinline__ uint32_t max_abs_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Zeros in place of bf16 elements that are not finite.
__device__ __forceinline__ void finite_only(uint32_t (&a)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if ((a[j] & 0x7f80u) == 0x7f80u) a[j] &= 0xffff0000u;
    if ((a[j] & 0x7f800000u) == 0x7f800000u) a[j] &= 0xffffu;
  }
}
// Token of a (token, query head) row.
__device__ __forceinline__ int token_of(int r, int T, int G) {
  return T == 1 ? 0 : G == 1 ? r : (int)((uint32_t)r / (uint32_t)G);
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// CTAs per SM: two; three where a warp's state is small, a key's bytes are few and the warps have keys of their own (e4m3,
// D = 64: 496 items of 10 rows x 5775 keys 102 against 117 us with two; 104 items of 32 rows x 3185 keys 35 against 31).
__host__ __device__ constexpr int ctas_per_sm(int D, bool q8, int wr) { return D == 64 && q8 && wr == 1 ? 3 : 2; }
__host__ __device__ constexpr int keys_per_tile(int D, bool q8) { return D == 64 || q8 ? 128 : 64; }

template <int D, bool Q8, int NB, int WR>
struct Geo {
  static constexpr int RB = D * (Q8 ? 1 : 2);             // bytes of a cached row
  static constexpr int RS = RB < 128 ? RB : 128;          // bytes of a row of a sub-tile, the widest that a copy swizzles
  static constexpr int SUBS = RB / RS;                    // sub-tiles side by side
  static constexpr int KT = keys_per_tile(D, Q8);         // keys per tile
  static constexpr int SUB = KT * RS;                     // bytes of a sub-tile
  static constexpr int STAGE = 2 * KT * RB;               // K and V
  static constexpr int CTAS = ctas_per_sm(D, Q8, WR);     // per SM
  static constexpr int LAUNCH_REGS = CTAS == 3 ? 80 : 128;
  static constexpr int COMPUTE_REGS = 2 * LAUNCH_REGS - 24;
  static constexpr int STAGES = (CTAS == 3 ? (NB == 1 ? 65536 : 49152) : STAGE <= 16384 ? 81920 : 98304) / STAGE;
  static constexpr int SCALE_STAGE = Q8 ? KT * 2 : 0;
  // Queries come with an item's first tile where they are few; otherwise their readers load them.
  static constexpr int QROW = D * 2 + 16;                 // a row's bytes, padded so that eight rows differ in their banks
  static constexpr int Q_STAGE = WR == 1 ? 8 * NB * QROW : 0;
  static constexpr int Q_AT = STAGES * (STAGE + SCALE_STAGE);
  static constexpr int RING = Q_AT + STAGES * Q_STAGE;
  static constexpr int RW = 8 * NB;                       // rows per warp
  static constexpr int RC = RW * WR;                      // rows per CTA
  static constexpr bool TWO = !Q8 && WR == 1;             // weights as the sum of two bf16 numbers
  static constexpr int COST = WR == 1 ? 1 : KT == 128 ? 2 : 4;  // of an item beside its tiles, in tiles
  static constexpr int ML = 4 * RW * 2;                   // maxima and sums of the four warps' rows, floats; twice
  static constexpr int SMEM = RING + 2 * ML * 4 + 2 * STAGES * 8 + 16 + 1024;  // and the start's alignment
  static_assert(4 * RW * D * 4 <= STAGE, "the warps' accumulators are joined in a consumed tile");
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "what an SM has for that many CTAs");
};

// The swizzle of a sub-tile's row: what its 16-byte chunk numbers are XORed with (as the copies do).
template <int RS>
__device__ __forceinline__ int swizzle_of(int row) {
  return RS == 64 ? (row >> 1) & 3 : row & 7;
}

// A tile of an item: sequence, key head, row tile, tile of keys.
struct Cursor {
  int b, h, rt, tile, ntile, len;
  int next_len;  // of the sequence behind, fetched ahead
};

// Length of a sequence as the kernel uses it: inside the caller's bound and the table's.
__device__ __forceinline__ int length_of(const PagedAttnParams& p, int b) {
  const int n = p.lens[b];
  if (n > p.max_len && p.status) atomicCAS(p.status, 0, (int)DEV_BAD_INDEX);
  return min(max(n, 0), p.max_len);
}
template <int KT>
__device__ __forceinline__ int tiles_of(int len) {
  return max(1, (len + KT - 1) / KT);
}

// The length of the sequence behind `b`, for advance().
__device__ __forceinline__ void look_ahead(const PagedAttnParams& p, Cursor& c) {
  c.next_len = c.b + 1 < p.B ? length_of(p, c.b + 1) : 0;
}

// All items lie on a line that the CTAs share evenly, each with COST units and one unit per tile behind them: what an item
// costs beside its tiles counts too, or a CTA over many short sequences would be the last by far (64 sequences of 0 to 2521
// keys x 16 heads, e4m3, head dimension 64: 66 us without, 50 with one unit, 53 with four; 16 sequences of 0 to 4121 keys x
// 35 rows x 4 heads, bf16: 37, 34 and 30 us, 31 with seven).  A CTA takes the tiles whose units lie in its range; every warp
// works that out for itself, by prefix sums over the sequences, a few per lane.
struct Range {
  int64_t total;       // units
  int64_t item_start;  // unit of the first tile of the item at the range's start
  int nc, nt;          // CTAs that have units, tiles of this one
};
__device__ __forceinline__ int64_t range_start(int64_t total, int nc, int c) {
  return total < 1 << 20 ? (int64_t)((uint32_t)total * (uint32_t)c / (uint32_t)nc) : total * c / nc;  // c <= nc < 2^12
}
__device__ __forceinline__ uint32_t divide(int64_t x, uint32_t d) {
  return (uint64_t)x >> 32 ? (uint32_t)((uint64_t)x / d) : (uint32_t)x / d;
}

// The first tile at or behind unit x, the unit of its item's first tile, and the number of tiles in front of x; by a warp
// whose lanes hold the sequences b0 .. b1 - 1 that begin at unit `at`.
template <int KT, int COST>
__device__ __forceinline__ int64_t locate(const PagedAttnParams& p, int64_t x, int64_t at, int64_t end, int b0, Cursor& cur,
                                          int64_t& item_start) {
  const int HR = p.Hkv * p.RT;
  int b = 0, len = 0;
  const bool here = x >= at && x < end;
  if (here) {
    for (b = b0;; ++b) {
      len = length_of(p, b);
      const int64_t next = at + (int64_t)(tiles_of<KT>(len) + COST) * HR;
      if (x < next) break;
      at = next;
    }
  }
  const int from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
  cur.b = __shfl_sync(0xffffffffu, b, from);
  cur.len = __shfl_sync(0xffffffffu, len, from);
  at = __shfl_sync(0xffffffffu, at, from);
  cur.ntile = tiles_of<KT>(cur.len);
  const uint32_t item = divide(x - at, (uint32_t)(cur.ntile + COST));
  const int64_t begin = at + (int64_t)item * (cur.ntile + COST) + COST;
  cur.tile = max((int)(x - begin), 0);
  cur.h = (int)(item / (uint32_t)p.RT);
  cur.rt = (int)(item - (uint32_t)cur.h * (uint32_t)p.RT);
  item_start = begin;
  return at - (int64_t)COST * HR * cur.b + (int64_t)item * cur.ntile + cur.tile;
}

template <int KT, int COST>
__device__ __forceinline__ Range warp_range(const PagedAttnParams& p, int ctas, int c, Cursor& cur) {
  const int lane = threadIdx.x & 31;
  const int per = (p.B + 31) / 32, b0 = min(lane * per, p.B), b1 = min(b0 + per, p.B);
  const int HR = p.Hkv * p.RT;
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += (int64_t)(tiles_of<KT>(length_of(p, b)) + COST) * HR;
  int64_t inc = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += x;
  }
  Range r;
  r.total = __shfl_sync(0xffffffffu, inc, 31);
  r.nc = (int)(r.total < ctas ? r.total : ctas);
  r.nt = 0;
  r.item_start = 0;
  cur = Cursor{};
  if (c >= r.nc) return r;
  const int64_t start = range_start(r.total, r.nc, c), end = range_start(r.total, r.nc, c + 1);
  int64_t behind = r.total - (int64_t)COST * HR * p.B, unused;
  if (end < r.total) behind = locate<KT, COST>(p, end, inc - mine, inc, b0, cur, unused);
  r.nt = (int)(behind - locate<KT, COST>(p, start, inc - mine, inc, b0, cur, r.item_start));
  look_ahead(p, cur);
  return r;
}
template <int KT>
__device__ __forceinline__ void advance(const PagedAttnParams& p, Cursor& c) {
  if (++c.tile < c.ntile) return;
  c.tile = 0;
  if (++c.rt < p.RT) return;
  c.rt = 0;
  if (++c.h < p.Hkv) return;
  c.h = 0;
  ++c.b;
  c.len = c.next_len;
  c.ntile = tiles_of<KT>(c.len);
  look_ahead(p, c);
}

// One warp's running state over an item.  Rows lie along the matrix instruction's 8 columns: a thread has the two rows
// 2 (lane mod 4) + {0, 1} of every block of 8, and of D the elements that element_of() gives.
template <int D, int NB>
struct State {
  float acc[D / 16][NB][4];  // [0], [1]: the two rows at a tile's first element of D, [2], [3]: at its second
  // scores in log2 units: this thread's maximum, the reference of its part `l` of the sum of exp2(s - ref) and, in bf16, of
  // the accumulators; e4m3: the same of score + V exponent, the reference of the accumulators
  float mx[NB][2], ref[NB][2], l[NB][2];
  float tmx[NB][2], tref[NB][2];
};
template <int D, bool RAW8>
__device__ __forceinline__ int element_of(int tile, int second) {
  const int g = (threadIdx.x & 31) >> 2;
  return RAW8 ? g * (D / 8) + 2 * tile + second : tile * 16 + 8 * second + g;
}

// Waits for a stage by a whole warp, with one answer for all lanes: false where the wait ran out.  With a limit of zero a
// phase that is not complete at the first look fails: mbar_wait's first look may itself be held for some microseconds.
__device__ __forceinline__ bool stage_wait(uint64_t* bar, uint32_t phase, const WaitCtx& w, int code) {
  bool ok = mbar_test_wait(bar, phase);
  if (!ok) {
    if (w.limit_ns == 0) {
      if (w.status) atomicCAS(w.status, 0, (int)DEV_FORCED_TIMEOUT);
      *w.abort_flag = 1;
    } else {
      ok = mbar_wait(bar, phase, w, code);
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// Fetches the tiles of a CTA's range, `nt` from `cur` on, into the ring.
template <class X, int D, bool Q8>
__device__ __forceinline__ void loader(const CUtensorMap& mk, const CUtensorMap& mv, const PagedAttnParams& p, Cursor cur, int nt,
                                       uint8_t* ring, uint64_t* full, uint64_t* empty, const WaitCtx& w) {
  const int lane = threadIdx.x & 31;
  const int box = 1 << p.box_log2;
  const uint32_t box_bytes = (uint32_t)box * (2 * X::RB + (Q8 ? 2 : 0));
  int stage = 0, issued = 0;
  uint32_t phase = 0;
  // this lane's box of a tile: how many boxes the tile has, the box's row in its page, the page (fetched a tile ahead)
  int boxes, row, page;
  auto look_up = [&](const Cursor& c) {
    const int key0 = c.tile * X::KT;
    boxes = min(X::KT >> p.box_log2, (c.len - key0 + box - 1) >> p.box_log2);  // 0 for an empty sequence
    const uint32_t grp = (uint32_t)(key0 + (lane << p.box_log2)) >> 4, pg = page_of_group(p.c, grp);
    row = (int)(grp - pg * p.c.groups) * 16;
    page = lane < boxes ? p.c.table[c.b * p.c.t_sb + pg] : 0;
  };
  if (nt > 0) look_up(cur);  // a CTA behind the line's end has no tile, and its cursor no sequence
  for (; issued < nt; ++issued) {
    Cursor next = cur;
    advance<X::KT>(p, next);
    const int now = boxes, now_row = row;
    int now_page = page;
    if (issued + 1 < nt) look_up(next);
    // A stage is filled again only when all four warps have seen its last tile arrive and have let go of it: no barrier is
    // armed while bytes of its phase before are under way.
    if (issued >= X::STAGES && !stage_wait(&empty[stage], phase ^ 1, w, DEV_TIMEOUT_PRODUCER)) break;
    const int r0 = cur.rt * X::RC;
    const int queries = X::Q_STAGE && (issued == 0 || cur.tile == 0) ? min(X::RC, p.R - r0) : 0;
    if (lane == 0) mbar_arrive_expect_tx(&full[stage], now * box_bytes + queries * D * 2);
    __syncwarp();
    if (lane < now) {
      if ((uint32_t)now_page >= (uint32_t)p.c.num_pages) {
        if (p.status) atomicCAS(p.status, 0, (int)DEV_BAD_INDEX);
        now_page = 0;
      }
      uint8_t* dst = ring + stage * X::STAGE + (lane << p.box_log2) * X::RS;
#pragma unroll
      for (int s = 0; s < X::SUBS; ++s) {
        tma_load_4d(dst + s * X::SUB, &mk, &full[stage], s * 64, now_row, cur.h, now_page);
        tma_load_4d(dst + X::KT * X::RB + s * X::SUB, &mv, &full[stage], s * 64, now_row, cur.h, now_page);
      }
      if constexpr (Q8) {
        bulk_load(smem_u32(ring + X::STAGES * X::STAGE + stage * X::SCALE_STAGE + (lane << p.box_log2) * 2),
                  p.c.scales + now_page * p.c.s_sp + cur.h * p.c.s_sh + now_row * 2, box * 2, &full[stage]);
      }
    }
    if (lane < queries) {
      const int r = r0 + lane, t = token_of(r, p.T, p.G), head = cur.h * p.G + r - t * p.G;
      bulk_load(smem_u32(ring + X::Q_AT + stage * X::Q_STAGE + lane * X::QROW), p.q + cur.b * p.q_sb + head * p.q_sh + t * p.q_sl,
                D * 2, &full[stage]);
    }
    cur = next;
    if (++stage == X::STAGES) stage = 0, phase ^= 1;
  }
  // Shared memory must not go while a copy is in flight, also after a wait that ran out: the last copies into every stage.
  for (int i = issued > X::STAGES ? issued - X::STAGES : 0; i < issued; ++i) {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(&full[i % X::STAGES], (i / X::STAGES) & 1)) {
      if (globaltimer_ns() - t0 > LVAR_DEFAULT_WAIT_NS) {
        if (p.status) atomicCAS(p.status, 0, (int)DEV_TIMEOUT_DRAIN);
        break;
      }
    }
  }
}

// O^T += V^T P^T of one step, 16 keys at a time.  CLEAN: elements of V that are not finite are left out.
template <class X, int D, bool Q8, int NB, int NK, bool CLEAN>
__device__ __forceinline__ void weigh(State<D, NB>& st, const float (&sc)[NK][NB][4], uint32_t vs, int s0) {
  const int lane = threadIdx.x & 31, quad = lane & 3;
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    uint32_t b[NB][2], rest[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const float w0 = sc[k][nb][2 * y], w1 = sc[k][nb][2 * y + 1];
        const uint32_t two = Q8 ? pack_f16x2(w0, w1) : pack_bf16x2(w0, w1);
        b[nb][y] = transpose8(two);
        // what the rounding to bf16 left of the weights
        if constexpr (X::TWO)
          rest[nb][y] = transpose8(pack_bf16x2(w0 - __uint_as_float(two << 16), w1 - __uint_as_float(two & 0xffff0000u)));
      }
    }
    if constexpr (!Q8) {
      const uint32_t v0 = vs + (s0 + k * 16 + (lane & 7) + ((lane >> 4) << 3)) * X::RS + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
      uint32_t a[D / 16][4], most = 0;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        ldsm_x4_t((v0 ^ ((t & 3) << 5)) + (t >> 2) * X::SUB, a[t]);
        if constexpr (CLEAN) finite_only(a[t]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma_bf16(st.acc[t][nb], a[t], b[nb][0], b[nb][1]);
        if constexpr (X::TWO && !CLEAN)
#pragma unroll
          for (int j = 0; j < 4; ++j) most = max_abs_bf16x2(most, a[t][j]);
      }
      if constexpr (X::TWO) {
        // An infinity has its product above; a rest of zero or below would make NaN of it.
        if (!CLEAN && __any_sync(0xffffffffu, (((most & 0x7f807f80u) + 0x00800080u) & 0x80008000u) != 0))
#pragma unroll
          for (int t = 0; t < D / 16; ++t) finite_only(a[t]);
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma_bf16(st.acc[t][nb], a[t], rest[nb][0], rest[nb][1]);
      }
    } else {
      constexpr int W = D / 32;  // words per thread and key: D / 8 consecutive elements, lane / 4 says which
      const uint32_t r0 = vs + (s0 + k * 16 + quad * 2) * X::RS;
      uint32_t u[4][W];
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // keys 2 quad, 2 quad + 1, and both + 8
        const uint32_t r = r0 + ((j & 1) + (j >> 1) * 8) * X::RS;
        if constexpr (D == 128) {
          const uint4 x = lds128(r + (((lane >> 2) ^ (quad * 2 + (j & 1))) << 4));
          u[j][0] = x.x, u[j][1] = x.y, u[j][2] = x.z, u[j][3] = x.w;
        } else {
          const uint2 x = lds64(r + (((lane >> 3) ^ quad) << 4) + ((lane >> 2) & 1) * 8);
          u[j][0] = x.x, u[j][1] = x.y;
        }
        if constexpr (CLEAN) {
#pragma unroll
          for (int i = 0; i < W; ++i)
#pragma unroll
            for (int y = 0; y < 4; ++y)
              if (((u[j][i] >> (8 * y)) & 0x7fu) == 0x7fu) u[j][i] &= ~(0xffu << (8 * y));
        }
      }
#pragma unroll
      for (int i = 0; i < W; ++i) {
        uint32_t a[2][4];
        widen4(__byte_perm(u[0][i], u[1][i], 0x5140), a[0][0], a[0][1]);
        widen4(__byte_perm(u[0][i], u[1][i], 0x7362), a[1][0], a[1][1]);
        widen4(__byte_perm(u[2][i], u[3][i], 0x5140), a[0][2], a[0][3]);
        widen4(__byte_perm(u[2][i], u[3][i], 0x7362), a[1][2], a[1][3]);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma_f16(st.acc[i * 2 + j][nb], a[j], b[nb][0], b[nb][1]);
      }
    }
  }
}

// Whether any element of a step's first `rows` V rows is not finite; by the whole warp.
template <class X, bool Q8, int NS>
__device__ __forceinline__ bool any_odd(uint32_t vs, int s0, int rows) {
  const int lane = threadIdx.x & 31;
  uint32_t hit = 0;
#pragma unroll
  for (int s = 0; s < X::SUBS; ++s) {
#pragma unroll
    for (int i = 0; i < NS * X::RS / 512; ++i) {
      const uint4 x = lds128(vs + s * X::SUB + s0 * X::RS + i * 512 + lane * 16);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 4 && (i * 512 + lane * 16) / X::RS < rows; ++j)
        hit |= Q8 ? ((w[j] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u : ((w[j] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
    }
  }
  return __any_sync(0xffffffffu, hit != 0);
}

// O^T += V^T P^T of a step with elements of V that are not finite: without them, and then row by row those that a row sees.
template <class X, int D, bool Q8, int NB, int NK>
__device__ __noinline__ void weigh_odd(State<D, NB>& st, const float (&sc)[NK][NB][4], const int (&seen)[NB][2], uint32_t vs,
                                       int s0) {
  weigh<X, D, Q8, NB, NK, true>(st, sc, vs, s0);
  const int quad = threadIdx.x & 3;
  for (int j = 0; j < NK * 16; ++j) {
    const int row = s0 + j, from = ((j & 7) << 2) | quad;  // the lane that has these rows' weights of key j
    for (int nb = 0; nb < NB; ++nb)
      for (int e = 0; e < 2; ++e) {
        const float w = __shfl_sync(0xffffffffu, sc[j >> 4][nb][((j >> 3) & 1) * 2 + e], from);
        for (int t = 0; t < D / 16; ++t)
          for (int second = 0; second < 2; ++second) {
            const int byte = element_of<D, Q8>(t, second) * (Q8 ? 1 : 2), chunk = (byte % X::RS) >> 4;
            const uint32_t at = vs + byte / X::RS * X::SUB + row * X::RS + ((chunk ^ swizzle_of<X::RS>(row)) << 4) + (byte & 15);
            const uint32_t bits = lds32(at & ~3u) >> ((at & 3u) * 8);
            const float val = Q8 ? NAN : __uint_as_float(bits << 16);
            const bool odd = Q8 ? (bits & 0x7fu) == 0x7fu : (bits & 0x7f80u) == 0x7f80u;
            float& acc = st.acc[t][nb][second * 2 + e];
            if (odd && j < seen[nb][e]) acc = fmaf(w, val, acc);
          }
      }
  }
}

__device__ __forceinline__ float max_of_keys(float x) {  // over the eight lanes that have the same rows
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
}
__device__ __forceinline__ float sum_of_keys(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 4);
  x += __shfl_xor_sync(0xffffffffu, x, 8);
  return x + __shfl_xor_sync(0xffffffffu, x, 16);
}

// The rest of a computing warp's way, `tiles` from `c` on, after a wait that ran out: to the barriers at the items' ends,
// where the other warps wait for it.  It lets go of no stage any more: the copies into the one it did not wait for may be in
// flight, and the loader, which needs all four warps to fill a stage again, gives up in turn.
template <class X>
__device__ __forceinline__ void give_up(const PagedAttnParams& p, Cursor c, int tiles) {
  for (; tiles > 0; --tiles) {
    if (c.tile == c.ntile - 1 || tiles == 1) {
      compute_sync();
      compute_sync();
    }
    advance<X::KT>(p, c);
  }
}

template <int D, bool Q8, int NB, int WR>
__global__ void __launch_bounds__(kAllThreads, (Geo<D, Q8, NB, WR>::CTAS))
    paged_attn_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                      const __grid_constant__ PagedAttnParams p) {
  using X = Geo<D, Q8, NB, WR>;
  constexpr int WK = 4 / WR;              // warps that share a row tile and differ in their keys
  constexpr int KW = X::KT / WK;          // keys of a tile per warp
  constexpr int NS = WR == 1 ? (KW < 32 ? KW : 32) : KW < 64 ? KW : 64;  // keys per step
  constexpr int NK = NS / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t ring = smem_u32(smem);
  float* const ml_first = reinterpret_cast<float*>(smem + X::RING);
  float* ml = ml_first;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + X::RING + 2 * X::ML * 4);
  uint64_t* empty = full + X::STAGES;
  int* abort_flag = reinterpret_cast<int*>(empty + X::STAGES);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wr = warp % WR, wk = warp / WR, quad = lane & 3, g8 = lane >> 2;
  const WaitCtx wait{p.status, abort_flag, p.wait_limit_ns};

  if (tid == 0) {
    for (int i = 0; i < X::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&mk);
    tma_prefetch_desc(&mv);
  }
  __syncthreads();
  griddep_wait();
  if (p.split) griddep_launch_dependents();
  if (warp > 4) {
    setmaxnreg_dec<24>();
    return;
  }
  Cursor cons;
  Range range;
  if (p.split) {
    range = warp_range<X::KT, X::COST>(p, (int)gridDim.x, blockIdx.x, cons);
  } else {
    const uint32_t HR = p.Hkv * p.RT, in = blockIdx.x % HR;
    cons.b = (int)(blockIdx.x / HR);
    cons.h = (int)(in / (uint32_t)p.RT);
    cons.rt = (int)(in % (uint32_t)p.RT);
    cons.tile = cons.next_len = 0;
    cons.len = length_of(p, cons.b);
    cons.ntile = range.nt = tiles_of<X::KT>(cons.len);
    range.item_start = 0;
  }
  const int nt = range.nt;
  if (warp == 4) {
    setmaxnreg_dec<24>();
    loader<X, D, Q8>(mk, mv, p, cons, nt, smem, full, empty, wait);
    return;
  }
  setmaxnreg_inc<X::COMPUTE_REGS>();

  State<D, NB> st;
  uint32_t qf[D / 16][NB][2];
  float qs[NB][2];      // factor from the raw product to log2 units, per row
  int limit[NB][2];     // keys that the row sees
  int see_all = 0;      // keys that every row of the item sees
  const bool whole_first = cons.tile == 0;  // the CTA's first piece begins at its item's start
  bool first_piece = true, fresh = true;
  int4 head = make_int4(0, 0, 0, 0);
  int64_t item_unit = range.item_start;  // of the item's first tile, on the line
  int stage = 0;
  uint32_t phase = 0;

  for (int i = 0; i < nt; ++i) {
    const int rt = cons.rt, h = cons.h;
    if (X::Q_STAGE && !stage_wait(&full[stage], phase, wait, DEV_TIMEOUT_SOFTMAX)) {
      give_up<X>(p, cons, nt - i);
      break;
    }
    if (fresh) {
      fresh = false;
      see_all = p.causal ? cons.len - p.T + 1 : cons.len;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) st.acc[t][nb][0] = st.acc[t][nb][1] = st.acc[t][nb][2] = st.acc[t][nb][3] = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          st.mx[nb][e] = st.ref[nb][e] = st.tmx[nb][e] = st.tref[nb][e] = -INFINITY;
          st.l[nb][e] = 0.f;
          const int r = rt * X::RC + wr * X::RW + nb * 8 + quad * 2 + e;
          limit[nb][e] = r >= p.R ? 0 : p.causal ? cons.len - p.T + token_of(r, p.T, p.G) + 1 : cons.len;
          qs[nb][e] = p.scale_log2;
        }
        // the queries as the instruction's second operand: row lane / 4
        const int r = rt * X::RC + wr * X::RW + nb * 8 + g8;
        const bool live = r < p.R;
        const int t = live ? token_of(r, p.T, p.G) : 0, g = live ? r - t * p.G : 0;
        const __nv_bfloat16* src =
            X::Q_STAGE ? reinterpret_cast<const __nv_bfloat16*>(smem + X::Q_AT + stage * X::Q_STAGE + (nb * 8 + g8) * X::QROW)
                       : p.q + cons.b * p.q_sb + (int64_t)(h * p.G + g) * p.q_sh + t * p.q_sl;
        if constexpr (!Q8) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            qf[kk][nb][0] = live ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + quad * 2) : 0u;
            qf[kk][nb][1] = live ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + quad * 2 + 8) : 0u;
          }
        } else {
          // matrix step 4 i + s takes elements 16 (2 quad + i) + 4 s + {0..3} (D = 64: 16 quad + 4 s) from this thread
          constexpr int CH = D / 64;
          uint2 raw[D / 16];
          float most = 0.f;
          bool fine = true;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            raw[kk] = live ? *reinterpret_cast<const uint2*>(src + 16 * (CH * quad + kk / 4) + 4 * (kk % 4)) : make_uint2(0u, 0u);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t w[2] = {raw[kk].x, raw[kk].y};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float a = fabsf(__uint_as_float(w[j] << 16)), b = fabsf(__uint_as_float(w[j] & 0xffff0000u));
              fine = fine && a < INFINITY && b < INFINITY;
              most = fmaxf(most, fmaxf(a, b));
            }
          }
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
          const int ex = min(max((int)(__float_as_uint(most) >> 23) - 127, -126), 126);
          const unsigned fines = __ballot_sync(0xffffffffu, fine) >> (lane & 28);
          const int sh = (fines & 15u) == 15u && most > 0.f ? ex : 0;
          const float down = pow2i(-sh);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            qf[kk][nb][0] = pack_f16x2(__uint_as_float(raw[kk].x << 16) * down, __uint_as_float(raw[kk].x & 0xffff0000u) * down);
            qf[kk][nb][1] = pack_f16x2(__uint_as_float(raw[kk].y << 16) * down, __uint_as_float(raw[kk].y & 0xffff0000u) * down);
          }
          // this thread's scores are those of rows 2 quad + e, scaled by lane 4 (2 quad + e)
#pragma unroll
          for (int e = 0; e < 2; ++e) qs[nb][e] *= pow2i(__shfl_sync(0xffffffffu, sh, (quad * 2 + e) * 4));
        }
      }
    }
    if (!X::Q_STAGE && !stage_wait(&full[stage], phase, wait, DEV_TIMEOUT_SOFTMAX)) {
      give_up<X>(p, cons, nt - i);
      break;
    }

    const bool idle = rt * X::RC + wr * X::RW >= p.R;  // none of the warp's rows exists
    const uint32_t ks = ring + stage * X::STAGE, vs = ks + X::KT * X::RB;
    const uint32_t ss = ring + X::STAGES * X::STAGE + stage * X::SCALE_STAGE;
#pragma unroll 1
    for (int s0 = wk * KW; s0 < (wk + 1) * KW; s0 += NS) {
      const int key0 = cons.tile * X::KT + s0;
      if (key0 >= cons.len || idle) break;  // the same for the whole warp
      const int rows = cons.len - key0;  // of the step's keys
      if (rows < NS) {
        // V rows behind the sequence's end become zeros: what a copy brought along or an earlier tile left may be anything
#pragma unroll
        for (int s = 0; s < X::SUBS; ++s)
          for (int at = rows * X::RS + lane * 16; at < NS * X::RS; at += 512) sts128(vs + s * X::SUB + s0 * X::RS + at, 0, 0, 0, 0);
        __syncwarp();
      }
      // scores, transposed: a thread has keys lane / 4 and + 8 of every 16, two rows of every 8
      float sc[NK][NB][4];
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) sc[k][nb][0] = sc[k][nb][1] = sc[k][nb][2] = sc[k][nb][3] = 0.f;
      if constexpr (!Q8) {
        const uint32_t k0 = ks + (s0 + (lane & 15)) * X::RS + (((lane >> 4) ^ (lane & 7)) << 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
          for (int k = 0; k < NK; ++k) {
            uint32_t a[4];
            ldsm_x4((k0 ^ ((kk & 3) << 5)) + (kk >> 2) * X::SUB + k * 16 * X::RS, a);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) mma_bf16(sc[k][nb], a, qf[kk][nb][0], qf[kk][nb][1]);
          }
        }
      } else {
        constexpr int CH = D / 64;
        const uint32_t k0 = ks + (s0 + g8) * X::RS + (((CH * quad) ^ swizzle_of<X::RS>(g8)) << 4);
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {
#pragma unroll
          for (int k = 0; k < NK; ++k) {
            const uint4 w0 = lds128((k0 ^ (ch << 4)) + k * 16 * X::RS), w1 = lds128((k0 ^ (ch << 4)) + (k * 16 + 8) * X::RS);
            const uint32_t u0[4] = {w0.x, w0.y, w0.z, w0.w}, u1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              uint32_t a[4];
              widen4(u0[s], a[0], a[2]);
              widen4(u1[s], a[1], a[3]);
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) mma_f16(sc[k][nb], a, qf[ch * 4 + s][nb][0], qf[ch * 4 + s][nb][1]);
            }
          }
        }
      }
      // e4m3: scores to log2 units, with the rows' scales (bf16: one factor, taken in with the maximum below)
      float ve[NK][2];  // V's exponents of the thread's keys
      if constexpr (Q8) {
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t ex = lds16(ss + (s0 + k * 16 + y * 8 + g8) * 2);  // K's, V's
            const float kf = __uint_as_float((ex << 23) & 0x7f800000u);
            ve[k][y] = __uint_as_float(0x4b000000u | (ex >> 8)) - (8388608.f + 127.f);  // 2^23 + byte, exact
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
              unpack_f32x2(fmul2(pack_f32x2(sc[k][nb][2 * y], sc[k][nb][2 * y + 1]),
                                 fmul2(pack_f32x2(kf, kf), pack_f32x2(qs[nb][0], qs[nb][1]))),
                           sc[k][nb][2 * y], sc[k][nb][2 * y + 1]);
          }
      }
      const bool edge = key0 + NS > see_all;  // some row does not see some of these keys
      if (edge) {
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key0 + k * 16 + (e >> 1) * 8 + g8 >= limit[nb][e & 1]) sc[k][nb][e] = -INFINITY;
      }
      // Weights relative to a reference that a row's scores have exceeded by at most 2^8: it moves to the maximum only when
      // they would, which is rare after an item's first step and spares every other one the exchange between lanes.
      bool grown = false;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float raw = -INFINITY;
#pragma unroll
          for (int k = 0; k < NK; ++k) {
            raw = fmax3(raw, sc[k][nb][e], sc[k][nb][2 + e]);
            if constexpr (Q8) st.tmx[nb][e] = fmax3(st.tmx[nb][e], sc[k][nb][e] + ve[k][0], sc[k][nb][2 + e] + ve[k][1]);
          }
          st.mx[nb][e] = fmaxf(st.mx[nb][e], Q8 ? raw : raw * qs[nb][e]);
          grown = grown || st.mx[nb][e] > st.ref[nb][e] + 8.f;
          if constexpr (Q8) grown = grown || st.tmx[nb][e] > st.tref[nb][e] + 8.f;
        }
      if (__any_sync(0xffffffffu, grown)) {
        float alpha[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            st.mx[nb][e] = max_of_keys(st.mx[nb][e]);
            float f = st.mx[nb][e] == -INFINITY ? 1.f : fast_exp2(st.ref[nb][e] - st.mx[nb][e]);
            st.l[nb][e] *= f;
            st.ref[nb][e] = st.mx[nb][e];
            if constexpr (Q8) {
              st.tmx[nb][e] = max_of_keys(st.tmx[nb][e]);
              f = st.tmx[nb][e] == -INFINITY ? 1.f : fast_exp2(st.tref[nb][e] - st.tmx[nb][e]);
              st.tref[nb][e] = st.tmx[nb][e];
            }
            alpha[nb][e] = f;
          }
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int y = 0; y < 2; ++y)
              unpack_f32x2(fmul2(pack_f32x2(st.acc[t][nb][2 * y], st.acc[t][nb][2 * y + 1]), pack_f32x2(alpha[nb][0], alpha[nb][1])),
                           st.acc[t][nb][2 * y], st.acc[t][nb][2 * y + 1]);
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float mu[2], tu[2];  // nothing seen so far: scores stay -inf
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mu[e] = st.ref[nb][e] == -INFINITY ? 0.f : -st.ref[nb][e];
          if constexpr (Q8) tu[e] = st.tref[nb][e] == -INFINITY ? 0.f : kUp - st.tref[nb][e];
        }
        uint64_t add = pack_f32x2(st.l[nb][0], st.l[nb][1]);
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint64_t s = pack_f32x2(sc[k][nb][2 * y], sc[k][nb][2 * y + 1]);
            float a, b;
            if constexpr (Q8) {
              unpack_f32x2(fadd2(s, pack_f32x2(mu[0], mu[1])), a, b);
              add = fadd2(add, pack_f32x2(fast_exp2(a), fast_exp2(b)));
              unpack_f32x2(fadd2(fadd2(s, pack_f32x2(ve[k][y], ve[k][y])), pack_f32x2(tu[0], tu[1])), a, b);
              sc[k][nb][2 * y] = fast_exp2(a);
              sc[k][nb][2 * y + 1] = fast_exp2(b);
            } else {
              unpack_f32x2(ffma2(s, pack_f32x2(qs[nb][0], qs[nb][1]), pack_f32x2(mu[0], mu[1])), a, b);
              sc[k][nb][2 * y] = fast_exp2(a);
              sc[k][nb][2 * y + 1] = fast_exp2(b);
              add = fadd2(add, pack_f32x2(sc[k][nb][2 * y], sc[k][nb][2 * y + 1]));
            }
          }
        unpack_f32x2(add, st.l[nb][0], st.l[nb][1]);
      }
      // In a step that some row does not see all of, elements of V that are not finite come in row by row: a weight of zero
      // would make NaN of them in rows that do not see them.
      if (edge && any_odd<X, Q8, NS>(vs, s0, rows)) {
        State<D, NB> st2 = st;
        float w[NK][NB][4];
        int seen[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
          for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) w[k][nb][e] = sc[k][nb][e];
          seen[nb][0] = limit[nb][0] - key0;
          seen[nb][1] = limit[nb][1] - key0;
        }
        weigh_odd<X, D, Q8, NB, NK>(st2, w, seen, vs, s0);
        st = st2;
      } else {
        weigh<X, D, Q8, NB, NK, false>(st, sc, vs, s0);
      }
    }

    const bool last = cons.tile == cons.ntile - 1;
    if (last || i == nt - 1) {
      // Join of the warps that share rows, in the stage just consumed.
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float m = max_of_keys(st.mx[nb][e]), l = sum_of_keys(st.l[nb][e]);
          if (g8 == 0)
            *reinterpret_cast<float2*>(ml + (warp * X::RW + nb * 8 + quad * 2 + e) * 2) =
                make_float2(m, m == -INFINITY ? 0.f : l * fast_exp2(st.ref[nb][e] - m));
        }
      compute_sync();
      // [warp][row][D]; elements are XORed with 8 times bits 1 and 2 of the row, so that a warp's rows differ in their banks
      float* buf = reinterpret_cast<float*>(smem + stage * X::STAGE);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = nb * 8 + quad * 2 + e;
          float top = -INFINITY;
#pragma unroll
          for (int w = 0; w < WK; ++w) top = fmaxf(top, ml[((w * WR + wr) * X::RW + row) * 2]);
          // an infinite maximum (an infinite score) gives NaN here, as exp(inf - inf) does
          const float own = Q8 ? st.tref[nb][e] - kUp : st.ref[nb][e];
          const float f = own == -INFINITY ? 0.f : fast_exp2(own - top);
          float* dst = buf + (warp * X::RW + row) * D;
          if constexpr (!Q8) {
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
              dst[element_of<D, false>(t, 0) ^ (quad * 8)] = st.acc[t][nb][e] * f;
              dst[element_of<D, false>(t, 1) ^ (quad * 8)] = st.acc[t][nb][2 + e] * f;
            }
          } else {
#pragma unroll
            for (int t = 0; t < D / 16; t += 2)
              *reinterpret_cast<float4*>(dst + (element_of<D, true>(t, 0) ^ (quad * 8))) = make_float4(
                  st.acc[t][nb][e] * f, st.acc[t][nb][2 + e] * f, st.acc[t + 1][nb][e] * f, st.acc[t + 1][nb][2 + e] * f);
          }
        }
      compute_sync();
      const bool whole = last && (!first_piece || whole_first);
      const int slot = first_piece ? 0 : 1;
      constexpr int TPR = D / 8, RPP = kThreads / TPR;
      const int e0 = (tid % TPR) * 8;
      const int live = min(X::RC, p.R - rt * X::RC);
#pragma unroll 4
      for (int row = tid / TPR; row < live; row += RPP) {
        const int w0 = row / X::RW, in = row % X::RW, ex = e0 ^ ((in >> 1 & 3) * 8);
        float top = -INFINITY, sum = 0.f, v[8] = {};
#pragma unroll
        for (int w = 0; w < WK; ++w) top = fmaxf(top, ml[((w * WR + w0) * X::RW + in) * 2]);
#pragma unroll
        for (int w = 0; w < WK; ++w) {
          const int at = (w * WR + w0) * X::RW + in;
          const float mw = ml[at * 2];
          sum += WK == 1 ? ml[at * 2 + 1] : mw == -INFINITY ? 0.f : ml[at * 2 + 1] * fast_exp2(mw - top);
          const float4 x = *reinterpret_cast<const float4*>(buf + at * D + ex);
          const float4 y = *reinterpret_cast<const float4*>(buf + at * D + ex + 4);
          v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
          v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
        }
        if (whole) {
          const int r = rt * X::RC + row, t = token_of(r, p.T, p.G), head = h * p.G + r - t * p.G;
          const float inv = top == -INFINITY ? 0.f : 1.f / sum;  // a row that sees no key gives 0
          uint4 out;
          out.x = pack_bf16x2(v[0] * inv, v[1] * inv);
          out.y = pack_bf16x2(v[2] * inv, v[3] * inv);
          out.z = pack_bf16x2(v[4] * inv, v[5] * inv);
          out.w = pack_bf16x2(v[6] * inv, v[7] * inv);
          *reinterpret_cast<uint4*>(p.o + cons.b * p.o_sb + head * p.o_sh + t * p.o_sl + e0) = out;
          if (p.M && e0 == 0) {
            const int64_t at = ((int64_t)cons.b * p.Hkv * p.G + head) * p.T + t;
            p.M[at] = top;
            p.L[at] = sum;
          }
        } else {
          float* dst = p.part + ((int64_t)blockIdx.x * kSlotsPerCta + slot) * (X::RC * (D + 2));
          *reinterpret_cast<float4*>(dst + row * D + e0) = make_float4(v[0], v[1], v[2], v[3]);
          *reinterpret_cast<float4*>(dst + row * D + e0 + 4) = make_float4(v[4], v[5], v[6], v[7]);
          if (e0 == 0) *reinterpret_cast<float2*>(dst + X::RC * D + row * 2) = make_float2(top, sum);
        }
      }
      if (!last && (!first_piece || whole_first)) {  // the head of an item that later CTAs go on with
        // the CTA whose range holds the unit of its last tile
        const int64_t end_tile = item_unit + cons.ntile - 1;
        int to = (int)(end_tile * range.nc / range.total);
        while (range_start(range.total, range.nc, to + 1) <= end_tile) ++to;
        while (range_start(range.total, range.nc, to) > end_tile) --to;
        head = make_int4(cons.b, cons.h * p.RT + rt, to - (int)blockIdx.x + 1, slot);
      }
      first_piece = false;
      fresh = true;
      ml = ml_first + (ml == ml_first ? X::ML : 0);  // a slow warp may still read this item's
      fence_proxy_async_smem();                      // the stage is written before the next copy into it
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[stage]);
    if (++stage == X::STAGES) stage = 0, phase ^= 1;
    if (last) item_unit += cons.ntile + X::COST;
    advance<X::KT>(p, cons);
  }
  if (p.split && tid == 0) p.heads[blockIdx.x] = head;
}

// Joins the pieces of the item that begins in CTA x's range and goes on behind it, in a fixed order.  Eight pieces of a row
// are under way at a time: the kernel is a chain of few memory latencies.
constexpr int kJoinWarps = 8;

template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const __grid_constant__ PagedAttnParams p, int rc) {
  constexpr int E = D / 32, BATCH = 8;
  __shared__ float sums[kJoinWarps][D], row_max[kJoinWarps], row_sum[kJoinWarps];
  const int c = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  griddep_wait();
  const int4 it = p.heads[c];
  const int n = it.z;
  if (n == 0) return;
  const int rt = it.y % p.RT, h = it.y / p.RT, rows = min(rc, p.R - rt * rc);
  const int64_t slot_floats = rc * (D + 2);
  // the first piece lies in the CTA's slot it.w, every later one in slot 0 of its CTA
  const float* first = p.part + ((int64_t)c * kSlotsPerCta + it.w) * slot_floats;
  const float* later = p.part + (int64_t)c * kSlotsPerCta * slot_floats;
  // Few pieces: a warp takes a row by itself; many: the CTA's warps share a row's pieces.
  const bool shared = n > 2 * BATCH;
  const int ways = shared ? kJoinWarps : 1, step = shared ? gridDim.y : gridDim.y * kJoinWarps;
  for (int row = shared ? blockIdx.y : blockIdx.y * kJoinWarps + warp; row < rows; row += step) {
    float top = -INFINITY, sum = 0.f, acc[E] = {};
    for (int i0 = shared ? warp : 0; i0 < n; i0 += ways * BATCH) {
      float2 x[BATCH];
      float v[BATCH][E];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int i = i0 + u * ways;
        x[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int e = 0; e < E; ++e) v[u][e] = 0.f;
        if (i < n) {
          const float* s = i == 0 ? first : later + (int64_t)i * kSlotsPerCta * slot_floats;
          x[u] = *reinterpret_cast<const float2*>(s + rc * D + row * 2);
          if constexpr (E == 4) {
            const float4 y = *reinterpret_cast<const float4*>(s + row * D + lane * E);
            v[u][0] = y.x, v[u][1] = y.y, v[u][2] = y.z, v[u][3] = y.w;
          } else {
            const float2 y = *reinterpret_cast<const float2*>(s + row * D + lane * E);
            v[u][0] = y.x, v[u][1] = y.y;
          }
        }
      }
      float next = top;
#pragma unroll
      for (int u = 0; u < BATCH; ++u) next = fmaxf(next, x[u].x);
      const float keep = top == -INFINITY ? 0.f : fast_exp2(top - next);
      sum *= keep;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= keep;
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const float f = x[u].x == -INFINITY ? 0.f : fast_exp2(x[u].x - next);
        sum = fmaf(x[u].y, f, sum);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(f, v[u][e], acc[e]);
      }
      top = next;
    }
    if (shared) {
#pragma unroll
      for (int e = 0; e < E; ++e) sums[warp][lane * E + e] = acc[e];
      if (lane == 0) row_max[warp] = top, row_sum[warp] = sum;
      __syncthreads();
      if (warp == 0) {
        top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, row_max[w]);
        sum = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) {
          const float f = row_max[w] == -INFINITY ? 0.f : fast_exp2(row_max[w] - top);
          sum = fmaf(row_sum[w], f, sum);
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] = fmaf(sums[w][lane * E + e], f, acc[e]);
        }
      }
      __syncthreads();
      if (warp != 0) continue;
    }
    const int r = rt * rc + row, t = token_of(r, p.T, p.G), head = h * p.G + r - t * p.G;
    const float inv = top == -INFINITY ? 0.f : 1.f / sum;  // a row that sees no key gives 0
    __nv_bfloat16* dst = p.o + it.x * p.o_sb + head * p.o_sh + t * p.o_sl + lane * E;
    if constexpr (E == 4) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
    } else {
      *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    }
    if (p.M && lane == 0) {
      const int64_t at = ((int64_t)it.x * p.Hkv * p.G + head) * p.T + t;
      p.M[at] = top;
      p.L[at] = sum;
    }
  }
}

// What a call launches: blocks of 8 rows per warp, warps that differ in their rows, row tiles, whether items are split, the
// number of CTAs.
struct Plan {
  int nb, wr, rt, split, ctas;
  int64_t workspace;
};

int device_sms(int* sms) {
  int dev = 0;
  LVAR_CUDA_OK(cudaGetDevice(&dev));
  LVAR_CUDA_OK(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
  return LVAR_OK;
}

int plan_of(int B, int Hq, int Hkv, int T, int D, bool q8, int max_len, int sms, Plan* out) {
  const int64_t R = (int64_t)T * (Hq / Hkv);
  out->nb = R <= 8 ? 1 : 2;
  out->wr = R <= 16 ? 1 : R <= 32 ? 2 : 4;
  const int rc = 8 * out->nb * out->wr;
  const int64_t rt = (R + rc - 1) / rc;
  const int kt = keys_per_tile(D, q8);
  const int64_t tiles = max_len <= kt ? 1 : ((int64_t)max_len + kt - 1) / kt;
  const int64_t items = B * (int64_t)Hkv * rt;
  LVAR_REQUIRE(items < (1ll << 24), LVAR_ERR_LIMIT, "too many (sequence, key head, row tile) items");
  out->rt = (int)rt;
  // Whether items are split.  A split costs the second kernel and a longer start, as much as `spare` tiles of an item take one
  // after the other; without it the longest item's tiles count, whatever the others have.  Where all items are under way at
  // once that is worth it while the tiles that a CTA would be spared are at most `spare`, taking the lengths to be half the
  // bound on average (bf16, D = 128, keys: 32 items 256: 6.6 against 8.6 us split, 512: 9.5 / 9.1; 256 items 256: 7.4 / 13.0,
  // 512: 10.6 / 15.4, 1024: 24.4 / 30.5; e4m3, 64 rows, 32 items 512: 21.2 / 21.1).  With more items a CTA per item pays for
  // its start each time (1024 items, bf16 128: 19.9 / 18.9, e4m3 512: 36.9 / 34.3), least where rows are many.
  const int64_t slots = (int64_t)ctas_per_sm(D, q8, out->wr) * sms, spare = out->wr == 4 && kt == 128 ? 4 : 6;
  out->split = items <= slots ? tiles * (2 * slots - items) > 2 * spare * slots : tiles > (out->wr == 1 ? 2 : spare);
  out->ctas = (int)(out->split ? slots : items);
  out->workspace = out->split ? (int64_t)out->ctas * (kSlotsPerCta * rc * (D + 2) * 4 + 16) : 0;
  return LVAR_OK;
}

template <int D, bool Q8, int NB, int WR>
int launch(const PagedAttnParams& p, const CUtensorMap& mk, const CUtensorMap& mv, const Plan& plan, cudaStream_t stream) {
  using X = Geo<D, Q8, NB, WR>;
  auto kern = paged_attn_kernel<D, Q8, NB, WR>;
  LVAR_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, X::SMEM));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)plan.ctas);
  cfg.blockDim = dim3(kAllThreads);
  cfg.dynamicSmemBytes = X::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LVAR_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, mk, mv, p));
  if (plan.split) {
    const int rows = p.R < X::RC ? p.R : X::RC;
    cfg.gridDim = dim3((unsigned)plan.ctas, (unsigned)(rows < 8 ? rows : 8));
    cfg.blockDim = dim3(kJoinWarps * 32);
    cfg.dynamicSmemBytes = 0;
    LVAR_CUDA_OK(cudaLaunchKernelEx(&cfg, paged_join_kernel<D>, p, X::RC));
  }
  return LVAR_OK;
}

template <int D, bool Q8>
int launch_wr(PagedAttnParams& p, const lvar_paged_cache& c, const Plan& plan, cudaStream_t stream) {
  const int KT = keys_per_tile(D, Q8);
  // Rows per copy: what page and tile have in common, and not far more than the longest sequence has.
  int box = KT;
  while (c.page_size % box != 0 || KT % box != 0) box -= 16;
  while (box % 32 == 0 && box / 2 >= p.max_len) box /= 2;
  p.box_log2 = 31 - __builtin_clz(box);  // a divisor of 64 or 128
  CUtensorMap mk, mv;
  if (int rc = encode_pages_map(&mk, c.k, Q8, c.num_pages, c.Hkv, c.page_size, D, c.k_sp, c.k_sh, c.k_sl, box)) return rc;
  if (int rc = encode_pages_map(&mv, c.v, Q8, c.num_pages, c.Hkv, c.page_size, D, c.v_sp, c.v_sh, c.v_sl, box)) return rc;
  if (plan.nb == 1) return launch<D, Q8, 1, 1>(p, mk, mv, plan, stream);
  if (plan.wr == 1) return launch<D, Q8, 2, 1>(p, mk, mv, plan, stream);
  if (plan.wr == 2) return launch<D, Q8, 2, 2>(p, mk, mv, plan, stream);
  return launch<D, Q8, 2, 4>(p, mk, mv, plan, stream);
}

}  // namespace

int64_t paged_attn_workspace(int B, int Hq, int Hkv, int T, int D, int q8, int max_len) {
  if (B < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv != 0 || T < 1 || max_len < 0 || max_len > 1 << 30 || (D != 64 && D != 128) ||
      (int64_t)T * Hq >= (1ll << 31))
    return fail(LVAR_ERR_ARG, "bad sizes");
  int sms = 0;
  if (int rc = device_sms(&sms)) return rc;
  Plan plan;
  if (int rc = plan_of(B, Hq, Hkv, T, D, q8 != 0, max_len, sms, &plan)) return rc;
  return plan.workspace;
}

int launch_paged_attn(const lvar_paged_attn_args* a, cudaStream_t stream) {
  LVAR_REQUIRE(a != nullptr, LVAR_ERR_ARG, "args must be non-null");
  PagedAttnParams p{};
  if (int rc = paged_view(&a->cache, &p.c)) return rc;
  const lvar_paged_cache& c = a->cache;
  LVAR_REQUIRE(a->q && a->o && a->lens, LVAR_ERR_ARG, "q, o and lens must be non-null");
  LVAR_REQUIRE((a->M == nullptr) == (a->L == nullptr), LVAR_ERR_ARG, "M and L go together");
  LVAR_REQUIRE(a->Hq >= 1 && a->T >= 1 && a->Hq % c.Hkv == 0, LVAR_ERR_ARG,
               "query heads must be a multiple of the cache's heads (got %d and %d)", a->Hq, c.Hkv);
  LVAR_REQUIRE((int64_t)a->T * a->Hq < (1ll << 31), LVAR_ERR_LIMIT, "too many query rows");
  LVAR_REQUIRE(a->scale > 0.f && a->scale < INFINITY, LVAR_ERR_ARG, "scale must be positive and finite");
  LVAR_REQUIRE(a->max_len >= 0 && a->max_len <= 1 << 30, LVAR_ERR_ARG, "max_len must lie in 0 .. 2^30");
  const int64_t strides[] = {a->q_sb, a->q_sh, a->q_sl, a->o_sb, a->o_sh, a->o_sl};
  for (int64_t s : strides)
    LVAR_REQUIRE(s >= 0 && s % 8 == 0, LVAR_ERR_ARG, "strides of q and o must be non-negative multiples of 8 elements");
  LVAR_REQUIRE(aligned16(a->q) && aligned16(a->o), LVAR_ERR_ARG, "q and o must be 16-byte aligned");
  const int64_t room = (int64_t)c.max_pages * c.page_size;
  const int max_len = (int)(a->max_len < room ? a->max_len : room);
  int sms = 0;
  if (int rc = device_sms(&sms)) return rc;
  Plan plan;
  if (int rc = plan_of(c.B, a->Hq, c.Hkv, a->T, c.D, c.scales != nullptr, a->max_len, sms, &plan)) return rc;
  LVAR_REQUIRE(plan.workspace == 0 || (a->workspace && aligned16(a->workspace) && a->workspace_bytes >= plan.workspace),
               LVAR_ERR_ARG, "workspace must be 16-byte aligned and hold %lld bytes (got %lld)", (long long)plan.workspace,
               (long long)a->workspace_bytes);
  p.lens = a->lens;
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.q_sb = a->q_sb; p.q_sh = a->q_sh; p.q_sl = a->q_sl;
  p.o = static_cast<__nv_bfloat16*>(a->o);
  p.o_sb = a->o_sb; p.o_sh = a->o_sh; p.o_sl = a->o_sl;
  p.M = a->M; p.L = a->L;
  p.part = static_cast<float*>(a->workspace);
  p.heads = reinterpret_cast<int4*>(p.part + (int64_t)plan.ctas * kSlotsPerCta * 8 * plan.nb * plan.wr * (c.D + 2));
  p.status = a->dev_status;
  p.B = c.B; p.Hkv = c.Hkv; p.G = a->Hq / c.Hkv; p.T = a->T; p.R = a->T * p.G;
  p.RT = plan.rt;
  p.causal = a->causal != 0; p.max_len = max_len;
  p.split = plan.split;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.wait_limit_ns = a->wait_limit_ns;
  if (c.D == 128) return c.scales ? launch_wr<128, true>(p, c, plan, stream) : launch_wr<128, false>(p, c, plan, stream);
  return c.scales ? launch_wr<64, true>(p, c, plan, stream) : launch_wr<64, false>(p, c, plan, stream);
}

}  // namespace lvar
