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

// A warp takes one token and 32 / (C / 8) * U of its rows (q heads, then k heads, then v heads).
template <int C, bool HALVES, bool Q8, int U>
__global__ void __launch_bounds__(256) paged_write_kernel(const __grid_constant__ WriteParams p, int units, int chunks) {
  constexpr int LPR = C / 8, RPW = 32 / LPR;
  const int lane = threadIdx.x & 31;
  const int unit = (int)blockIdx.x * 8 + (int)(threadIdx.x >> 5);
  if (unit >= units) return;
  const int t = unit / chunks, b = t / p.L, l = t - b * p.L;
  const int g = lane / LPR, x = lane % LPR;
  const int e0 = HALVES ? x * 4 : x * 8;
  constexpr int kHigh = HALVES ? C / 2 : 4;  // where a lane's elements 4..7 begin, from its element 0
  const int rows = p.Hq + 2 * p.Hkv;
  const int r0 = (unit - t * chunks) * (RPW * U) + g;
  const bool there = p.count == nullptr || l < p.count[b];

  uint2 raw[U][2];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int r = r0 + u * RPW;
    raw[u][0] = raw[u][1] = make_uint2(0u, 0u);
    if (r < rows && there) {
      const int kind = r < p.Hq ? 0 : r < p.Hq + p.Hkv ? 1 : 2;
      const int h = kind == 0 ? r : kind == 1 ? r - p.Hq : r - p.Hq - p.Hkv;
      const __nv_bfloat16* src = p.x[kind] + b * p.s_b[kind] + l * p.s_l[kind] + h * p.s_h[kind] + e0;
      if constexpr (HALVES) {
        raw[u][0] = *reinterpret_cast<const uint2*>(src);
        raw[u][1] = *reinterpret_cast<const uint2*>(src + kHigh);
      } else {
        const uint4 w = *reinterpret_cast<const uint4*>(src);
        raw[u][0] = make_uint2(w.x, w.y);
        raw[u][1] = make_uint2(w.z, w.w);
      }
    }
  }
  const int first = p.start[b];
  const int pos = first < 0 || first > kMaxTokens ? -1 : first + l;
  Place at{-1, 0};
  if (there && r0 + (U - 1) * RPW >= p.Hq) at = place_of(p.c, b, pos, p.status);
  float cs[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {};
  if (p.cos_t != nullptr && there) {
    if ((uint32_t)pos >= (uint32_t)p.rope_rows && p.status) atomicCAS(p.status, 0, (int)DEV_BAD_INDEX);
    const int64_t row = min(max(pos, 0), p.rope_rows - 1);
    const float4 c4 = __ldg(reinterpret_cast<const float4*>(p.cos_t + row * (C / 2) + x * 4));
    const float4 s4 = __ldg(reinterpret_cast<const float4*>(p.sin_t + row * (C / 2) + x * 4));
    cs[0] = c4.x, cs[1] = c4.y, cs[2] = c4.z, cs[3] = c4.w;
    sn[0] = s4.x, sn[1] = s4.y, sn[2] = s4.z, sn[3] = s4.w;
  }

#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int r = r0 + u * RPW;
    const int kind = r < p.Hq ? 0 : r < p.Hq + p.Hkv ? 1 : 2;
    const int h = kind == 0 ? r : kind == 1 ? r - p.Hq : r - p.Hq - p.Hkv;
    const uint32_t w[4] = {raw[u][0].x, raw[u][0].y, raw[u][1].x, raw[u][1].y};
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    if (p.norm != 0) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
#pragma unroll
      for (int d = LPR / 2; d >= 1; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
      if (kind < 2 && r < rows) {
        if (p.norm == 1) {
          const float f = __frcp_rn(fmaxf(sqrtf(ss), 1e-12f)), m = kind == 0 ? p.scale_mul[h] : 1.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = v[e] * f * m;
        } else {
          const float f = rsqrtf(ss * (1.f / C) + p.eps);
          const float* wt = kind == 0 ? p.wq : p.wk;
          if (wt != nullptr) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(wt + e0));
            const float4 c = __ldg(reinterpret_cast<const float4*>(wt + e0 + kHigh));
            const float wv[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = v[e] * f * wv[e];
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= f;
          }
        }
      }
    }
    if (p.cos_t != nullptr && kind < 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ia = HALVES ? i : 2 * i, ib = HALVES ? i + 4 : 2 * i + 1;
        const float a = v[ia], c = v[ib];
        v[ia] = fmaf(cs[i], a, -(sn[i] * c));
        v[ib] = fmaf(sn[i], a, cs[i] * c);
      }
    }
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = kind == 2 ? w[i] : pack_bf16x2(v[2 * i], v[2 * i + 1]);
    float most = 0.f;
    if constexpr (Q8) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = fabsf(v[e]);
        most = fmaxf(most, a < INFINITY ? a : 0.f);
      }
#pragma unroll
      for (int d = LPR / 2; d >= 1; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
    }
    if (r >= rows) continue;
    if (kind == 0) {
      __nv_bfloat16* dst = p.q_out + b * p.q_sb + h * p.q_sh + l * p.q_sl + e0;  // rows of padding are 0
      if constexpr (HALVES) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
        *reinterpret_cast<uint2*>(dst + kHigh) = make_uint2(o[2], o[3]);
      } else {
        *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    } else if (at.page >= 0) {
      uint8_t* base = kind == 1 ? p.c.k + at.page * p.c.k_sp + h * p.c.k_sh + at.row * p.c.k_sl
                                : p.c.v + at.page * p.c.v_sp + h * p.c.v_sh + at.row * p.c.v_sl;
      if constexpr (!Q8) {
        if constexpr (HALVES) {
          *reinterpret_cast<uint2*>(base + e0 * 2) = make_uint2(o[0], o[1]);
          *reinterpret_cast<uint2*>(base + (e0 + kHigh) * 2) = make_uint2(o[2], o[3]);
        } else {
          *reinterpret_cast<uint4*>(base + e0 * 2) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      } else {
        // most = s * 2^q with 1 <= s < 2: 448 = 1.75 * 2^8, so e = q - 8, and one more where s > 1.75
        const uint32_t bits = __float_as_uint(most);
        int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
        e = most == 0.f ? -100 : min(max(e, -100), 120);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fabsf(v[i]) < INFINITY ? v[i] * down : NAN;
        const uint32_t lo = narrow4(v[0], v[1], v[2], v[3]), hi = narrow4(v[4], v[5], v[6], v[7]);
        if constexpr (HALVES) {
          *reinterpret_cast<uint32_t*>(base + e0) = lo;
          *reinterpret_cast<uint32_t*>(base + e0 + kHigh) = hi;
        } else {
          *reinterpret_cast<uint2*>(base + e0) = make_uint2(lo, hi);
        }
        if (x == 0) p.c.scales[at.page * p.c.s_sp + h * p.c.s_sh + at.row * 2 + (kind - 1)] = (uint8_t)(e + 127);
      }
    }
  }
}

template <int C, bool HALVES, bool Q8, int U>
int launch_write_u(const WriteParams& p, cudaStream_t stream) {
  constexpr int ROWS = 32 / (C / 8) * U;
  const int64_t rows = (int64_t)p.Hq + 2ll * p.Hkv;
  const int64_t chunks = (rows + ROWS - 1) / ROWS, units = (int64_t)p.B * p.L * chunks;
  LVAR_REQUIRE(units < (1ll << 31) - 8, LVAR_ERR_LIMIT, "too many rows");
  paged_write_kernel<C, HALVES, Q8, U><<<(unsigned)((units + 7) / 8), 256, 0, stream>>>(p, (int)units, (int)chunks);
  LVAR_CUDA_OK(cudaGetLastError());
  return LVAR_OK;
}
template <int C, bool HALVES, bool Q8>
int launch_write_q(const WriteParams& p, cudaStream_t stream) {
  const int64_t units = (int64_t)p.B * p.L * (((int64_t)p.Hq + 2ll * p.Hkv) * (C / 8) / 128);
  return units >= 2 * 148 * 40 ? launch_write_u<C, HALVES, Q8, 4>(p, stream) : launch_write_u<C, HALVES, Q8, 1>(p, stream);
}
template <int C>
int launch_write_c(const WriteParams& p, bool halves, cudaStream_t stream) {
  if (p.c.scales) return halves ? launch_write_q<C, true, true>(p, stream) : launch_write_q<C, false, true>(p, stream);
  return halves ? launch_write_q<C, true, false>(p, stream) : launch_write_q<C, false, false>(p, stream);
}

struct ReadParams {
  PagedView c;
  const int32_t* lens;
  __nv_bfloat16* o[2];
  int64_t o_sb[2], o_sh[2], o_sl[2];
  int32_t* status;
  int B, Hkv, start, n, blocks;  // blocks per (sequence, head)
};

// Eight elements per lane.  A CTA takes U * 256 / (D / 8) rows of one (sequence, head), K and V.
template <int D, bool Q8, int U>
__global__ void __launch_bounds__(256) paged_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int LPR = D / 8, RPB = 256 / LPR;
  const int bh = blockIdx.x / p.blocks, blk = blockIdx.x - bh * p.blocks;
  const int b = bh / p.Hkv, h = bh - b * p.Hkv;
  const int x = threadIdx.x % LPR, r0 = blk * (RPB * U) + threadIdx.x / LPR;
  const int len = min(p.lens[b], kMaxTokens);
  uint4 w[U][2];
  uint32_t ex[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = r0 + u * RPB;
    const int pos = p.start + i;
    w[u][0] = w[u][1] = make_uint4(0u, 0u, 0u, 0u);
    ex[u] = 0;
    if (i >= p.n || pos >= len) continue;
    const Place at = place_of(p.c, b, pos, p.status);
    if (at.page < 0) continue;
    const uint8_t* kr = p.c.k + at.page * p.c.k_sp + h * p.c.k_sh + at.row * p.c.k_sl;
    const uint8_t* vr = p.c.v + at.page * p.c.v_sp + h * p.c.v_sh + at.row * p.c.v_sl;
    if constexpr (Q8) {
      const uint2 a = *reinterpret_cast<const uint2*>(kr + x * 8), c = *reinterpret_cast<const uint2*>(vr + x * 8);
      w[u][0].x = a.x, w[u][0].y = a.y;
      w[u][1].x = c.x, w[u][1].y = c.y;
      ex[u] = *reinterpret_cast<const uint16_t*>(p.c.scales + at.page * p.c.s_sp + h * p.c.s_sh + at.row * 2);
    } else {
      w[u][0] = *reinterpret_cast<const uint4*>(kr + x * 16);
      w[u][1] = *reinterpret_cast<const uint4*>(vr + x * 16);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = r0 + u * RPB;
    if (i >= p.n) continue;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      uint4 out = w[u][y];
      if constexpr (Q8) {
        const float up = __uint_as_float(((ex[u] >> (8 * y)) & 0xffu) << 23);
        const uint32_t in[2] = {w[u][y].x, w[u][y].y};
        uint32_t r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t two = in[j >> 1] >> (16 * (j & 1));
          uint32_t f16;
          asm("{\n.reg .b16 t;\ncvt.u16.u32 t, %1;\ncvt.rn.f16x2.e4m3x2 %0, t;\n}" : "=r"(f16) : "r"(two));
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&f16));
          r[j] = pack_bf16x2(f.x * up, f.y * up);
        }
        out = make_uint4(r[0], r[1], r[2], r[3]);
      }
      *reinterpret_cast<uint4*>(p.o[y] + b * p.o_sb[y] + h * p.o_sh[y] + i * p.o_sl[y] + x * 8) = out;
    }
  }
}

template <int D, bool Q8, int U>
int launch_read_u(ReadParams p, cudaStream_t stream) {
  constexpr int ROWS = 256 / (D / 8) * U;
  p.blocks = (p.n + ROWS - 1) / ROWS;
  const int64_t grid = (int64_t)p.B * p.Hkv * p.blocks;
  LVAR_REQUIRE(grid < (1ll << 31), LVAR_ERR_LIMIT, "too many rows");
  paged_read_kernel<D, Q8, U><<<(unsigned)grid, 256, 0, stream>>>(p);
  LVAR_CUDA_OK(cudaGetLastError());
  return LVAR_OK;
}
template <int D, bool Q8>
int launch_read_q(const ReadParams& p, cudaStream_t stream) {
  const int64_t blocks = (int64_t)p.B * p.Hkv * p.n / (256 / (D / 8) * 4);
  return blocks >= 148 * 8 ? launch_read_u<D, Q8, 4>(p, stream) : launch_read_u<D, Q8, 1>(p, stream);
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
  LVAR_REQUIRE((int64_t)c.B * a->L < (1ll << 31), LVAR_ERR_LIMIT, "too many tokens");
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
  for (int64_t s : strides)
    LVAR_REQUIRE(s >= 0 && s % 8 == 0, LVAR_ERR_ARG, "strides must be non-negative multiples of 8 elements");
  LVAR_REQUIRE(aligned16(a->k) && aligned16(a->v), LVAR_ERR_ARG, "tensors must be 16-byte aligned");
  p.lens = a->lens;
  p.o[0] = static_cast<__nv_bfloat16*>(a->k);
  p.o[1] = static_cast<__nv_bfloat16*>(a->v);
  p.o_sb[0] = a->k_sb; p.o_sh[0] = a->k_sh; p.o_sl[0] = a->k_sl;
  p.o_sb[1] = a->v_sb; p.o_sh[1] = a->v_sh; p.o_sl[1] = a->v_sl;
  p.status = a->dev_status;
  p.B = c.B; p.Hkv = c.Hkv; p.start = a->start; p.n = a->n;
  if (c.D == 128) return c.scales ? launch_read_q<128, true>(p, stream) : launch_read_q<128, false>(p, stream);
  return c.scales ? launch_read_q<64, true>(p, stream) : launch_read_q<64, false>(p, stream);
}

}  // namespace lvar
