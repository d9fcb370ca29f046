// Writing and reading the paged key/value cache.
//
// paged_write_kernel: rows of new tokens go to the cache at position start[b] + l, as they are (append) or after the
// prologue of a self-attention layer: norms of q and k over the head dimension and the position rotation,
//   L2:  x / max(|x|, 1e-12), q also times scale_mul[h]      RMS: x * rsqrt(mean x^2 + eps) * weight[e]
//   rotation by the angle of (position, i): pairs (2i, 2i+1), or (i, i + c/2) with `halves`
// all in fp32 on the widened bf16 inputs, rounded once: q and a bf16 cache to bf16, an e4m3 cache to the row's scale
//   2^e, e the least integer with max |x| 2^-e <= 448, -100 <= e <= 120   (elements that are not finite become NaN and
//   do not take part in the maximum; a row of zeros has e = -100).
// A power of two makes the row's widening exact (an e4m3 times 2^e is a bf16 number) and costs no accuracy: e4m3 keeps 4
// bits of significand whatever the scale.
// Bound by HBM (2 c bytes in and 2 c or c + 1 out per token and head) once a call is large, by latency below.  c / 8 lanes
// share a row and hold 8 elements each; with `halves` a lane holds 4 elements of either half, so that a rotation's two
// elements are always in one lane.
//
// paged_read_kernel: rows start .. start + n of every sequence out of the pages as contiguous bf16, zeros behind a
// sequence's end: what the many-query attention kernels take.  One pass, bound by HBM.
#include <math.h>

#include "paged.cuh"
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace lvar {

int paged_view(const lvar_paged_cache* c, PagedView* out) {
  LVAR_REQUIRE(c->k && c->v && c->table, LVAR_ERR_ARG, "cache k, v and table must be non-null");
  LVAR_REQUIRE(c->D == 64 || c->D == 128, LVAR_ERR_UNSUPPORTED, "Head dimension must be 64 or 128 (got %d)", c->D);
  LVAR_REQUIRE(c->B >= 1 && c->Hkv >= 1 && c->num_pages >= 1 && c->max_pages >= 1, LVAR_ERR_ARG, "bad cache sizes");
  LVAR_REQUIRE(c->page_size >= 16 && c->page_size <= 512 && c->page_size % 16 == 0, LVAR_ERR_UNSUPPORTED,
               "page_size must be a multiple of 16 up to 512 (got %d)", c->page_size);
  const int elt = c->scales ? 1 : 2, mult = 16 / elt;
  const int64_t strides[] = {c->k_sp, c->k_sh, c->k_sl, c->v_sp, c->v_sh, c->v_sl};
  for (int64_t s : strides)
    LVAR_REQUIRE(s >= 0 && s % mult == 0, LVAR_ERR_ARG, "cache strides must be non-negative multiples of %d elements", mult);
  LVAR_REQUIRE(aligned16(c->k) && aligned16(c->v), LVAR_ERR_ARG, "cache tensors must be 16-byte aligned");
  if (c->scales) {
    LVAR_REQUIRE(c->s_sp >= 0 && c->s_sh >= 0 && c->s_sp % 16 == 0 && c->s_sh % 16 == 0 && aligned16(c->scales), LVAR_ERR_ARG,
                 "scales must be 16-byte aligned with page and head strides in multiples of 16");
  }
  LVAR_REQUIRE(c->t_sb >= 0, LVAR_ERR_ARG, "the table's stride must not be negative");
  PagedView v{};
  v.k = static_cast<uint8_t*>(c->k);
  v.v = static_cast<uint8_t*>(c->v);
  v.scales = c->scales;
  v.k_sp = c->k_sp * elt; v.k_sh = c->k_sh * elt; v.k_sl = c->k_sl * elt;
  v.v_sp = c->v_sp * elt; v.v_sh = c->v_sh * elt; v.v_sl = c->v_sl * elt;
  v.s_sp = c->s_sp; v.s_sh = c->s_sh;
  v.table = c->table;
  v.t_sb = c->t_sb;
  v.num_pages = c->num_pages;
  v.max_pages = c->max_pages;
  v.groups = (uint32_t)c->page_size / 16;
  v.magic = v.groups == 1 ? 0u : (uint32_t)(((1ull << 32) + v.groups - 1) / v.groups);
  *out = v;
  return LVAR_OK;
}

namespace {

constexpr int kMaxTokens = 1 << 30;  // positions stay below this

struct WriteParams {
  PagedView c;
  const __nv_bfloat16* x[3];  // q (or null), k, v
  int64_t s_b[3], s_l[3], s_h[3];
  const int32_t* start;
  const int32_t* count;  // or null: all L
  const float* scale_mul;
  const float* wq;
  const float* wk;
  const float* cos_t;
  const float* sin_t;
  __nv_bfloat16* q_out;
  int64_t q_sb, q_sh, q_sl;
  int32_t* status;
  float eps;
  int norm;  // 0 none, 1 L2, 2 RMS
  int rope_rows;
  int B, L, Hq, Hkv;
};

// Where a token's rows go: byte offsets of its page row, or page < 0 where it has none.
struct Place {
  int page;
  uint32_t row;
};
__device__ __forceinline__ Place place_of(const PagedView& c, int b, int pos, int32_t* status) {
  Place at{-1, 0};
  const uint32_t grp = (uint32_t)pos >> 4, pg = page_of_group(c, grp);
  if (pos >= 0 && pos < kMaxTokens && pg < (uint32_t)c.max_pages) {
    const int page = c.table[b * c.t_sb + pg];
    if ((uint32_t)page < (uint32_t)c.num_pages) {
      at.page = page;
      at.row = (grp - pg * c.groups) * 16 + (pos & 15);
    }
  }
  if (at.page < 0 && status) atomicCAS(status, 0, (int)DEV_BAD_INDEX);
  return at;
}

__device__ __forceinline__ uint32_t narrow4(float a, float b, float c, float d) {  // four e4m3 bytes, a lowest
  uint32_t r;
  asm("{\n.reg .b16 lo, hi;\ncvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\ncvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n"
      "mov.b32 %0, {lo, hi};\n}"
      : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

// Biased exponent of a row's scale: the least e with most * 2^-e <= 448 = 1.75 * 2^8, -100 <= e <= 120.  For most = s * 2^q
// with 1 <= s < 2 that is q - 8, and one more where s > 1.75: the addend carries into the exponent just then.  A maximum over
// nothing but NaN is NaN and counts as 0: fmaxf takes the number.
__device__ __forceinline__ int scale_byte(float most) {
  return min(max((int)((__float_as_uint(fmaxf(most, 0.f)) + 0x1fffffu) >> 23) - 8, 27), 247);
}

// A CTA's eight warps take a token each; a warp takes RPW * U rows of one kind (q, k or v heads), grid.y says which.  Where
// rows are only appended and a token has fewer heads than a warp takes, it takes 1 << tsh tokens (U = 1).
// A lane's eight elements are held as the first and the second elements of four rotations, two rotations in a 64-bit pair
// for packed arithmetic: with pairs (2i, 2i + 1) these are the halves of a 32-bit word, with `HALVES` four elements of either
// half of the row.  The rotation table is read once for the warp's rows; indices are 32-bit but for the final addresses.
// A row whose kind is decided row by row, with a library root, reciprocal and unpacked arithmetic, cost 210 instructions a
// lane and bound the kernel by issue: 52 us for 2 x 4096 tokens x 48 heads x 128, 38 us now (0.81 of the
// measured copy rate; two rows a lane instead of four 48 us).
// BARE: rows go without norm and rotation (to a bf16 cache: as they are).
template <int C, bool HALVES, bool Q8, bool BARE, int U>
__global__ void __launch_bounds__(256, BARE ? (Q8 ? 4 : 6) : 3) paged_write_kernel(const __grid_constant__ WriteParams p, int cq, int ck, int tsh) {
  constexpr int LPR = C / 8, RPW = 32 / LPR;
  const int lane = threadIdx.x & 31;
  constexpr int LOG_RPW = C == 128 ? 1 : 2;
  const int hsh = LOG_RPW - tsh, group = lane / LPR;
  const int token = (((int)blockIdx.x * 8 + (int)(threadIdx.x >> 5)) << tsh) + (group >> hsh);
  bool alive = token < p.B * p.L;
  if (!__any_sync(0xffffffffu, alive)) return;
  const int t = alive ? token : 0;
  const int b = (int)((uint32_t)t / (uint32_t)p.L), l = t - b * p.L;
  const int kind = (int)blockIdx.y < cq ? 0 : (int)blockIdx.y < cq + ck ? 1 : 2;
  const int chunk = (int)blockIdx.y - (kind == 0 ? 0 : kind == 1 ? cq : cq + ck);
  const int heads = kind == 0 ? p.Hq : p.Hkv;
  const int g = group & ((1 << hsh) - 1), x = lane % LPR;
  const int e0 = HALVES ? x * 4 : x * 8;
  constexpr int kHigh = HALVES ? C / 2 : 4;  // where a lane's elements 4..7 begin, from its element 0
  const int h0 = chunk * (RPW * U) + g;
  const bool there = alive && (p.count == nullptr || l < p.count[b]);

  const __nv_bfloat16* src = (kind == 0 ? p.x[0] + b * p.s_b[0] + l * p.s_l[0] + h0 * p.s_h[0]
                              : kind == 1 ? p.x[1] + b * p.s_b[1] + l * p.s_l[1] + h0 * p.s_h[1]
                                          : p.x[2] + b * p.s_b[2] + l * p.s_l[2] + h0 * p.s_h[2]) + e0;
  const int64_t step = RPW * (kind == 0 ? p.s_h[0] : kind == 1 ? p.s_h[1] : p.s_h[2]);
  uint2 raw[U][2];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    raw[u][0] = raw[u][1] = make_uint2(0u, 0u);
    if (h0 + u * RPW < heads && there) {
      if constexpr (HALVES) {
        raw[u][0] = *reinterpret_cast<const uint2*>(src);
        raw[u][1] = *reinterpret_cast<const uint2*>(src + kHigh);
      } else {
        const uint4 w = *reinterpret_cast<const uint4*>(src);
        raw[u][0] = make_uint2(w.x, w.y);
        raw[u][1] = make_uint2(w.z, w.w);
      }
    }
    src += step;
  }
  float mul[U];  // the heads' factors
#pragma unroll
  for (int u = 0; u < U; ++u) mul[u] = !BARE && kind == 0 && p.norm == 1 && h0 + u * RPW < heads ? __ldg(p.scale_mul + h0 + u * RPW) : 1.f;
  const int first = p.start[b];
  const int pos = first < 0 || first > kMaxTokens ? -1 : first + l;
  Place at{-1, 0};
  if (kind != 0) {
    if (there) at = place_of(p.c, b, pos, p.status);
    alive = at.page >= 0;  // else padding, or nowhere to go
    if (!__any_sync(0xffffffffu, alive)) return;
  }
  uint64_t cs[2], sn[2], ns[2];  // cosines and sines of the lane's four rotations, and the sines negated
  if (!BARE && p.cos_t != nullptr && kind < 2) {
    if (there && (uint32_t)pos >= (uint32_t)p.rope_rows && p.status) atomicCAS(p.status, 0, (int)DEV_BAD_INDEX);
    const int64_t row = min(max(pos, 0), p.rope_rows - 1);
    const float4 c4 = __ldg(reinterpret_cast<const float4*>(p.cos_t + row * (C / 2) + x * 4));
    const float4 s4 = __ldg(reinterpret_cast<const float4*>(p.sin_t + row * (C / 2) + x * 4));
    cs[0] = pack_f32x2(c4.x, c4.y), cs[1] = pack_f32x2(c4.z, c4.w);
    sn[0] = pack_f32x2(s4.x, s4.y), sn[1] = pack_f32x2(s4.z, s4.w);
    ns[0] = pack_f32x2(-s4.x, -s4.y), ns[1] = pack_f32x2(-s4.z, -s4.w);
  }
  const float* wt = !BARE && p.norm == 2 && kind < 2 ? (kind == 0 ? p.wq : p.wk) : nullptr;
  uint64_t wa[2], wb[2];  // norm weights of the first and second elements
  if (wt != nullptr) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(wt + e0)), c = __ldg(reinterpret_cast<const float4*>(wt + e0 + kHigh));
    wa[0] = HALVES ? pack_f32x2(a.x, a.y) : pack_f32x2(a.x, a.z), wb[0] = HALVES ? pack_f32x2(c.x, c.y) : pack_f32x2(a.y, a.w);
    wa[1] = HALVES ? pack_f32x2(a.z, a.w) : pack_f32x2(c.x, c.z), wb[1] = HALVES ? pack_f32x2(c.z, c.w) : pack_f32x2(c.y, c.w);
  }

  uint8_t* base = nullptr;
  int64_t out_step = 0;
  if (kind == 1) {
    base = p.c.k + at.page * p.c.k_sp + h0 * p.c.k_sh + at.row * p.c.k_sl;
    out_step = RPW * p.c.k_sh;
  } else if (kind == 2) {
    base = p.c.v + at.page * p.c.v_sp + h0 * p.c.v_sh + at.row * p.c.v_sl;
    out_step = RPW * p.c.v_sh;
  } else {
    base = reinterpret_cast<uint8_t*>(p.q_out + b * p.q_sb + h0 * p.q_sh + l * p.q_sl);
    out_step = RPW * p.q_sh * 2;
  }
  auto store = [&](int u, const uint32_t (&o)[4]) {
    if (h0 + u * RPW >= heads || !alive) return;
    uint8_t* dst = base + u * out_step;
    if constexpr (HALVES) {
      *reinterpret_cast<uint2*>(dst + e0 * 2) = make_uint2(o[0], o[1]);
      *reinterpret_cast<uint2*>(dst + (e0 + kHigh) * 2) = make_uint2(o[2], o[3]);
    } else {
      *reinterpret_cast<uint4*>(dst + e0 * 2) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  };
  if (kind == 0 && !there) {  // padding, the same for the whole warp
#pragma unroll
    for (int u = 0; u < U; ++u) store(u, {0u, 0u, 0u, 0u});
    return;
  }
  bool copy = kind == 2 && !Q8;
  if (BARE && !Q8) copy = true;
  if (copy) {  // as they are
#pragma unroll
    for (int u = 0; u < U; ++u) store(u, {raw[u][0].x, raw[u][0].y, raw[u][1].x, raw[u][1].y});
    return;
  }

  // Step by step for all rows, so that their chains of shuffles and roots overlap.
  uint64_t A[U][2], B[U][2];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t w[4] = {raw[u][0].x, raw[u][0].y, raw[u][1].x, raw[u][1].y};
    auto lo = [&](int i) { return __uint_as_float(w[i] << 16); };
    auto hi = [&](int i) { return __uint_as_float(w[i] & 0xffff0000u); };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      A[u][i] = HALVES ? pack_f32x2(lo(i), hi(i)) : pack_f32x2(lo(2 * i), lo(2 * i + 1));
      B[u][i] = HALVES ? pack_f32x2(lo(i + 2), hi(i + 2)) : pack_f32x2(hi(2 * i), hi(2 * i + 1));
    }
  }
  if (!BARE && kind < 2 && p.norm != 0) {
    float y[U], f[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float s0, s1;
      unpack_f32x2(ffma2(B[u][1], B[u][1], ffma2(B[u][0], B[u][0], ffma2(A[u][1], A[u][1], fmul2(A[u][0], A[u][0])))), s0, s1);
      y[u] = s0 + s1;
    }
#pragma unroll
    for (int d = LPR / 2; d >= 1; d >>= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) y[u] += __shfl_xor_sync(0xffffffffu, y[u], d);
    bool plain = true;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p.norm == 2) y[u] = fmaf(y[u], 1.f / C, p.eps);
      // the hardware's reciprocal root and one Newton step: half an ulp more than the nearest at most
      f[u] = rsqrtf(y[u]);
      f[u] = fmaf(0.5f * f[u], fmaf(-y[u] * f[u], f[u], 1.f), f[u]);
      plain = plain && y[u] > 1e-24f && y[u] < 1e38f;
    }
    if (!plain) {  // a norm that is clamped (by a comparison: a NaN stays one), zero or not finite
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (y[u] > 1e-24f && y[u] < 1e38f) continue;
        const float norm = sqrtf(y[u]);
        f[u] = 1.f / (p.norm == 1 && norm < 1e-12f ? 1e-12f : norm);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t ff = pack_f32x2(f[u] * mul[u], f[u] * mul[u]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        A[u][i] = fmul2(A[u][i], ff);
        B[u][i] = fmul2(B[u][i], ff);
      }
    }
    if (wt != nullptr) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          A[u][i] = fmul2(A[u][i], wa[i]);
          B[u][i] = fmul2(B[u][i], wb[i]);
        }
    }
  }
  if (!BARE && kind < 2 && p.cos_t != nullptr) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint64_t a = ffma2(B[u][i], ns[i], fmul2(A[u][i], cs[i]));
        B[u][i] = ffma2(B[u][i], cs[i], fmul2(A[u][i], sn[i]));
        A[u][i] = a;
      }
  }
  if (!Q8 || kind == 0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float a[4], c[4];
      unpack_f32x2(A[u][0], a[0], a[1]), unpack_f32x2(A[u][1], a[2], a[3]);
      unpack_f32x2(B[u][0], c[0], c[1]), unpack_f32x2(B[u][1], c[2], c[3]);
      if constexpr (HALVES) {
        store(u, {pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(c[0], c[1]), pack_bf16x2(c[2], c[3])});
      } else {
        store(u, {pack_bf16x2(a[0], c[0]), pack_bf16x2(a[1], c[1]), pack_bf16x2(a[2], c[2]), pack_bf16x2(a[3], c[3])});
      }
    }
    return;
  }
  // an 8-bit row
  float most[U];
  auto largest = [&](int u) {  // passes over NaN
    float a[4], c[4];
    unpack_f32x2(A[u][0], a[0], a[1]), unpack_f32x2(A[u][1], a[2], a[3]);
    unpack_f32x2(B[u][0], c[0], c[1]), unpack_f32x2(B[u][1], c[2], c[3]);
    return fmaxf(fmax3(fmax3(fabsf(a[0]), fabsf(a[1]), fabsf(a[2])), fabsf(a[3]), fabsf(c[0])),
                 fmax3(fabsf(c[1]), fabsf(c[2]), fabsf(c[3])));
  };
  bool endless = false;
#pragma unroll
  for (int u = 0; u < U; ++u) most[u] = largest(u);
#pragma unroll
  for (int d = LPR / 2; d >= 1; d >>= 1)
#pragma unroll
    for (int u = 0; u < U; ++u) most[u] = fmaxf(most[u], __shfl_xor_sync(0xffffffffu, most[u], d));
#pragma unroll
  for (int u = 0; u < U; ++u) endless = endless || most[u] == INFINITY;
  if (__any_sync(0xffffffffu, endless)) {  // infinities become NaN and the maximum is taken again
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float a, c;
        unpack_f32x2(A[u][i], a, c);
        A[u][i] = pack_f32x2(fabsf(a) < INFINITY ? a : NAN, fabsf(c) < INFINITY ? c : NAN);
        unpack_f32x2(B[u][i], a, c);
        B[u][i] = pack_f32x2(fabsf(a) < INFINITY ? a : NAN, fabsf(c) < INFINITY ? c : NAN);
      }
      most[u] = largest(u);
#pragma unroll
      for (int d = LPR / 2; d >= 1; d >>= 1) most[u] = fmaxf(most[u], __shfl_xor_sync(0xffffffffu, most[u], d));
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int byte = scale_byte(most[u]);
    const float down = __uint_as_float((uint32_t)(254 - byte) << 23);
    const uint64_t dd = pack_f32x2(down, down);
    float a[4], c[4];
    unpack_f32x2(fmul2(A[u][0], dd), a[0], a[1]), unpack_f32x2(fmul2(A[u][1], dd), a[2], a[3]);
    unpack_f32x2(fmul2(B[u][0], dd), c[0], c[1]), unpack_f32x2(fmul2(B[u][1], dd), c[2], c[3]);
    const int h = h0 + u * RPW;
    if (h >= heads || !alive) continue;
    uint8_t* dst = base + u * out_step;
    if constexpr (HALVES) {
      *reinterpret_cast<uint32_t*>(dst + e0) = narrow4(a[0], a[1], a[2], a[3]);
      *reinterpret_cast<uint32_t*>(dst + e0 + kHigh) = narrow4(c[0], c[1], c[2], c[3]);
    } else {
      *reinterpret_cast<uint2*>(dst + e0) = make_uint2(narrow4(a[0], c[0], a[1], c[1]), narrow4(a[2], c[2], a[3], c[3]));
    }
    if (x == 0) p.c.scales[at.page * p.c.s_sp + h * p.c.s_sh + at.row * 2 + (kind - 1)] = (uint8_t)byte;
  }
}

template <int C, bool HALVES, bool Q8, bool BARE, int U>
int launch_write_u(const WriteParams& p, cudaStream_t stream) {
  constexpr int ROWS = 32 / (C / 8) * U;
  const int cq = (p.Hq + ROWS - 1) / ROWS, ck = (p.Hkv + ROWS - 1) / ROWS;
  LVAR_REQUIRE((int64_t)cq + 2 * ck <= 65535, LVAR_ERR_LIMIT, "too many heads");
  int tsh = 0;
  if constexpr (U == 1) {  // 30 x 3752 tokens x 2 heads x 64 in bf16: 30 us against 43 with a token per warp
    if (p.Hq == 0)
      while ((32 / (C / 8) >> (tsh + 1)) >= p.Hkv) ++tsh;
  }
  const int64_t warps = ((int64_t)p.B * p.L + (1 << tsh) - 1) >> tsh;
  const dim3 grid((unsigned)((warps + 7) / 8), (unsigned)(cq + 2 * ck));
  paged_write_kernel<C, HALVES, Q8, BARE, U><<<grid, 256, 0, stream>>>(p, cq, ck, tsh);
  LVAR_CUDA_OK(cudaGetLastError());
  return LVAR_OK;
}
// Several rows per lane once one row each would fill the chip (148 SMs of 40 warps) twice over, as many as leave at most a quarter of the lanes
// without a row; one row otherwise: the shortest chain of dependent steps, which is all that a small call waits for.
template <int C, bool HALVES, bool Q8, bool BARE>
int launch_write_q(const WriteParams& p, cudaStream_t stream) {
  constexpr int RPW = 32 / (C / 8);
  const int64_t tokens = (int64_t)p.B * p.L, rows = (int64_t)p.Hq + 2ll * p.Hkv;
  auto padded = [&](int n) { return ((int64_t)(p.Hq + n - 1) / n + 2 * ((p.Hkv + n - 1) / n)) * n; };
  if (tokens * rows >= 2 * 148 * 40 * RPW) {
    if (4 * rows >= 3 * padded(4 * RPW)) return launch_write_u<C, HALVES, Q8, BARE, 4>(p, stream);
    if (4 * rows >= 3 * padded(2 * RPW)) return launch_write_u<C, HALVES, Q8, BARE, 2>(p, stream);
  }
  return launch_write_u<C, HALVES, Q8, BARE, 1>(p, stream);
}
template <int C>
int launch_write_c(const WriteParams& p, bool halves, cudaStream_t stream) {
  const bool bare = p.norm == 0 && p.cos_t == nullptr;  // the layout of rotations does not matter then
  if (bare) return p.c.scales ? launch_write_q<C, false, true, true>(p, stream) : launch_write_q<C, false, false, true>(p, stream);
  if (p.c.scales) return halves ? launch_write_q<C, true, true, false>(p, stream) : launch_write_q<C, false, true, false>(p, stream);
  return halves ? launch_write_q<C, true, false, false>(p, stream) : launch_write_q<C, false, false, false>(p, stream);
}

struct ReadParams {
  PagedView c;
  const int32_t* lens;
  __nv_bfloat16* o[2];
  int64_t o_sb[2], o_sh[2], o_sl[2];
  int32_t* status;
  int B, Hkv, start, n, blocks;  // blocks per (sequence, head)
  bool wide;                     // outputs start on 32-byte boundaries
};

// Four e4m3 bytes times a power of two as four bf16 (exact).
__device__ __forceinline__ uint2 widen_scaled(uint32_t four, uint64_t up) {
  uint32_t lo, hi;
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}"
      : "=r"(lo), "=r"(hi) : "r"(four));
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo)), y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  float a, b, c, d;
  unpack_f32x2(fmul2(pack_f32x2(x.x, x.y), up), a, b);
  unpack_f32x2(fmul2(pack_f32x2(y.x, y.y), up), c, d);
  return make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
}

// A lane reads 16 bytes of a row: 8 elements of a bf16 cache, 16 of an e4m3 one.  A CTA takes 256 / lanes-per-row rows of one
// (sequence, head), K and V (two or four rows per lane changed nothing: 43.9 us for 8 x 16 heads x 2521 e4m3 rows of 128,
// 0.87 of the measured copy rate).
template <int D, bool Q8>
__global__ void __launch_bounds__(256) paged_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int LPR = D * (Q8 ? 1 : 2) / 16, RPB = 256 / LPR;
  const int bh = blockIdx.x / p.blocks, blk = blockIdx.x - bh * p.blocks;
  const int b = bh / p.Hkv, h = bh - b * p.Hkv;
  const int x = threadIdx.x % LPR, i = blk * RPB + threadIdx.x / LPR;
  if (i >= p.n) return;
  uint4 w[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
  uint32_t ex = 0;
  if (p.start + i < min(p.lens[b], kMaxTokens)) {
    const Place at = place_of(p.c, b, p.start + i, p.status);
    if (at.page >= 0) {
      w[0] = *reinterpret_cast<const uint4*>(p.c.k + at.page * p.c.k_sp + h * p.c.k_sh + at.row * p.c.k_sl + x * 16);
      w[1] = *reinterpret_cast<const uint4*>(p.c.v + at.page * p.c.v_sp + h * p.c.v_sh + at.row * p.c.v_sl + x * 16);
      if constexpr (Q8) ex = *reinterpret_cast<const uint16_t*>(p.c.scales + at.page * p.c.s_sp + h * p.c.s_sh + at.row * 2);
    }
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    uint4* dst = reinterpret_cast<uint4*>(p.o[y] + b * p.o_sb[y] + h * p.o_sh[y] + i * p.o_sl[y] + x * (Q8 ? 16 : 8));
    if constexpr (Q8) {
      const float f = __uint_as_float(((ex >> (8 * y)) & 0xffu) << 23);
      const uint64_t up = pack_f32x2(f, f);
      const uint2 a = widen_scaled(w[y].x, up), c = widen_scaled(w[y].y, up);
      const uint2 d = widen_scaled(w[y].z, up), e = widen_scaled(w[y].w, up);
      if (p.wide) {  // a sector per lane; two 16-byte stores would write half sectors
        const uint32_t all[8] = {a.x, a.y, c.x, c.y, d.x, d.y, e.x, e.y};
        st_global_v8(dst, all);
      } else {
        dst[0] = make_uint4(a.x, a.y, c.x, c.y);
        dst[1] = make_uint4(d.x, d.y, e.x, e.y);
      }
    } else {
      dst[0] = w[y];
    }
  }
}

template <int D, bool Q8>
int launch_read(ReadParams p, cudaStream_t stream) {
  constexpr int ROWS = 256 / (D * (Q8 ? 1 : 2) / 16);
  p.blocks = (p.n + ROWS - 1) / ROWS;
  const int64_t grid = (int64_t)p.B * p.Hkv * p.blocks;
  LVAR_REQUIRE(grid < (1ll << 31), LVAR_ERR_LIMIT, "too many rows");
  paged_read_kernel<D, Q8><<<(unsigned)grid, 256, 0, stream>>>(p);
  LVAR_CUDA_OK(cudaGetLastError());
  return LVAR_OK;
}

}  // namespace

int launch_paged_write(const lvar_paged_write_args* a, cudaStream_t stream) {
  LVAR_REQUIRE(a != nullptr, LVAR_ERR_ARG, "args must be non-null");
  WriteParams p{};
  if (int rc = paged_view(&a->cache, &p.c)) return rc;
  const lvar_paged_cache& c = a->cache;
  LVAR_REQUIRE(a->k && a->v && a->start, LVAR_ERR_ARG, "k, v and start must be non-null");
  LVAR_REQUIRE((a->q == nullptr) == (a->Hq == 0) && (a->q == nullptr) == (a->q_out == nullptr) && a->Hq >= 0, LVAR_ERR_ARG,
               "q, q_out and Hq go together");
  LVAR_REQUIRE(a->L >= 1 && a->L <= kMaxTokens, LVAR_ERR_ARG, "bad number of tokens");
  LVAR_REQUIRE((int64_t)c.B * a->L <= kMaxTokens, LVAR_ERR_LIMIT, "too many tokens");
  LVAR_REQUIRE(a->norm >= 0 && a->norm <= 2, LVAR_ERR_ARG, "norm must be 0, 1 or 2");
  LVAR_REQUIRE(a->norm != 1 || a->scale_mul || a->Hq == 0, LVAR_ERR_ARG, "the L2 norm takes scale_mul");
  LVAR_REQUIRE(a->norm != 2 || a->eps >= 0.f, LVAR_ERR_ARG, "eps must not be negative");
  LVAR_REQUIRE((a->rope_cos == nullptr) == (a->rope_sin == nullptr), LVAR_ERR_ARG, "rope_cos and rope_sin go together");
  LVAR_REQUIRE(a->rope_cos == nullptr || a->rope_rows >= 1, LVAR_ERR_ARG, "the rotation tables have no rows");
  const int64_t strides[] = {a->q_sb, a->q_sl, a->q_sh, a->k_sb, a->k_sl, a->k_sh, a->v_sb, a->v_sl, a->v_sh,
                             a->qo_sb, a->qo_sh, a->qo_sl};
  for (int64_t s : strides)
    LVAR_REQUIRE(s >= 0 && s % 8 == 0, LVAR_ERR_ARG, "strides must be non-negative multiples of 8 elements");
  const void* ptrs[] = {a->q, a->k, a->v, a->q_out, a->rope_cos, a->rope_sin, a->q_weight, a->k_weight};
  for (const void* x : ptrs) LVAR_REQUIRE(aligned16(x), LVAR_ERR_ARG, "tensors must be 16-byte aligned");
  const void* xs[3] = {a->q, a->k, a->v};
  const int64_t sb[3] = {a->q_sb, a->k_sb, a->v_sb}, sl[3] = {a->q_sl, a->k_sl, a->v_sl}, sh[3] = {a->q_sh, a->k_sh, a->v_sh};
  for (int i = 0; i < 3; ++i) {
    p.x[i] = static_cast<const __nv_bfloat16*>(xs[i]);
    p.s_b[i] = sb[i]; p.s_l[i] = sl[i]; p.s_h[i] = sh[i];
  }
  p.start = a->start;
  p.count = a->count;
  p.scale_mul = a->scale_mul;
  p.wq = a->q_weight; p.wk = a->k_weight;
  p.cos_t = a->rope_cos; p.sin_t = a->rope_sin;
  p.q_out = static_cast<__nv_bfloat16*>(a->q_out);
  p.q_sb = a->qo_sb; p.q_sh = a->qo_sh; p.q_sl = a->qo_sl;
  p.status = a->dev_status;
  p.eps = a->eps;
  p.norm = a->norm;
  p.rope_rows = a->rope_rows;
  p.B = c.B; p.L = a->L; p.Hq = a->Hq; p.Hkv = c.Hkv;
  return c.D == 128 ? launch_write_c<128>(p, a->rope_halves != 0, stream) : launch_write_c<64>(p, a->rope_halves != 0, stream);
}

int launch_paged_read(const lvar_paged_read_args* a, cudaStream_t stream) {
  LVAR_REQUIRE(a != nullptr, LVAR_ERR_ARG, "args must be non-null");
  ReadParams p{};
  if (int rc = paged_view(&a->cache, &p.c)) return rc;
  const lvar_paged_cache& c = a->cache;
  LVAR_REQUIRE(a->k && a->v && a->lens, LVAR_ERR_ARG, "k, v and lens must be non-null");
  LVAR_REQUIRE(a->start >= 0 && a->n >= 1 && (int64_t)a->start + a->n <= kMaxTokens, LVAR_ERR_ARG, "bad row range");
  const int64_t strides[] = {a->k_sb, a->k_sh, a->k_sl, a->v_sb, a->v_sh, a->v_sl};
  p.wide = ((reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v)) & 31) == 0;
  for (int64_t s : strides) {
    LVAR_REQUIRE(s >= 0 && s % 8 == 0, LVAR_ERR_ARG, "strides must be non-negative multiples of 8 elements");
    p.wide = p.wide && s % 16 == 0;
  }
  LVAR_REQUIRE(aligned16(a->k) && aligned16(a->v), LVAR_ERR_ARG, "tensors must be 16-byte aligned");
  p.lens = a->lens;
  p.o[0] = static_cast<__nv_bfloat16*>(a->k);
  p.o[1] = static_cast<__nv_bfloat16*>(a->v);
  p.o_sb[0] = a->k_sb; p.o_sh[0] = a->k_sh; p.o_sl[0] = a->k_sl;
  p.o_sb[1] = a->v_sb; p.o_sh[1] = a->v_sh; p.o_sl[1] = a->v_sl;
  p.status = a->dev_status;
  p.B = c.B; p.Hkv = c.Hkv; p.start = a->start; p.n = a->n;
  if (c.D == 128) return c.scales ? launch_read<128, true>(p, stream) : launch_read<128, false>(p, stream);
  return c.scales ? launch_read<64, true>(p, stream) : launch_read<64, false>(p, stream);
}

}  // namespace lvar
