// New tokens into a paged 4-bit cache, with the norms of q and k per head and the rotation by
// position on the way, in one launch (sm_100a).
//
// Tokens come packed: token r of cu[b] .. cu[b + 1] - 1 is new token i = r - cu[b] of sequence b, at
// cache place lens[b] + i and position P = lens[b] + i + pos_offset[b].  Per row of 128 channels:
// x <- w x / sqrt(mean(x^2) + eps) (with weights), then the first `rot` channels are turned pairwise
// by P * inv_freq[j] (pairs (j, j + rot / 2), or (2j, 2j + 1) interleaved).  q' and k' are rounded
// once, to the model's type; K's codes are those of the unrounded k (paged4.cuh).
//
// Codes are those of exact arithmetic.  P * inv_freq is formed in float64 and taken as a fraction of
// a turn; norms and turns are float32, off by at most kSlack of |x cos| + |o sin|.  A row with a
// quotient or a scale closer to a rounding border than that (about 1 in 100) is formed again in
// float64.  V's codes come from its 16-bit values: an 11-bit x over an 11-bit s is 2^-13 away from a
// border unless it lies on it, and one corrected division finds both cases.
//
// Bound by memory: per token (Hq + 2 Hkv) rows read, Hq (+ Hkv) rows and Hkv 144 bytes written.  16
// lanes hold a row (8 channels, 16 bytes, each); a half-warp takes one token and all of its rows, two
// in flight.  cos and sin of a block's tokens are formed once, in shared memory.
#include <algorithm>

#include "paged4.cuh"

namespace hq {
int current_sm_count();

namespace p4 {

constexpr int kThreads = 128;
constexpr int kTok = kThreads / 16;       // tokens per block

struct AppendParams {
  Pages pg;
  const void* q;
  const void* k;
  const void* v;
  int64_t qs[2], ks[2], vs[2], qos[2], kos[2];  // element strides of token and head
  int T, B, Hq, Hkv;
  const int* cu;                          // null: token r is sequence r's only one
  const int* lens;
  const int* pos_offset;
  const void* qw;
  const void* kw;
  int w_f32;
  float eps;
  const float* inv_freq;
  int rot, inter;
  float factor;
  void* q_out;
  void* k_out;
  int copy_rest;                          // q_out takes q's rows behind the last sequence
  int* status;
  int rows_per_block, groups;
  float slack;
};

// Error of the float32 route, of |x w| + |o w_o|: half that of a sum of 128 squares (8 in a lane,
// 4 rounds: 12 x 2^-24) 2^-21.4, rsqrt 2^-22, cos and sin 2^-22.5 and their product with a weight
// 2^-24, the turn's roundings 2^-23.4 and r's product 2^-24: 2^-19.95 in all.
constexpr float kSlack = 1.0e-6f;

template <int DT>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (DT == HQ_DTYPE_BF16) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&x);
  } else {
    const __half2 x = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&x);
  }
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
// The scale of a group from amax / 7.5: NaN where amax is no number, the largest float16 above it.
__device__ __forceinline__ __half group_scale(float a75) {
  if (!(a75 < INFINITY)) return __ushort_as_half(0x7fff);
  return __float2half_rn(fminf(a75, 65504.0f));
}
// 8 rounded quotients as a word of nibbles
__device__ __forceinline__ uint32_t pack_codes(const float (&t)[8]) {
  float c[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = fminf(fmaxf(rintf(t[e]), -8.0f), 7.0f);
  // 4 codes as one whole number below 2^15 (c + 8 would cost an add each: 8 * 0x1111 at once)
  const float lo = __fmaf_rn(4096.0f, c[3], __fmaf_rn(256.0f, c[2], __fmaf_rn(16.0f, c[1], c[0])));
  const float hi = __fmaf_rn(4096.0f, c[7], __fmaf_rn(256.0f, c[6], __fmaf_rn(16.0f, c[5], c[4])));
  return static_cast<uint32_t>(static_cast<int>(lo) + 0x8888) |
         static_cast<uint32_t>(static_cast<int>(hi) + 0x8888) << 16;
}

// One k row in float64 (all 16 lanes of the half-warp `mask`): this lane's word and group's scale.
struct Exact {
  uint32_t word;
  __half scale;
};
template <int DT>
__device__ __noinline__ Exact exact_row(const AppendParams& p, const uint4& x, unsigned mask, int partner,
                                        double pos, int l) {
  float f[8];
  Vec16<DT>::unpack(x, f);
  const int d0 = 8 * l, half = p.rot / 2;
  double y[8], o[8], r = 1.0;
  if (p.kw) {
    double s = 0.0;
#pragma unroll 1
    for (int e = 0; e < 8; ++e) s += static_cast<double>(f[e]) * f[e];
#pragma unroll 1
    for (int m = 8; m >= 1; m >>= 1) s += __shfl_xor_sync(mask, s, m);
    r = 1.0 / sqrt(s / kD + static_cast<double>(p.eps));
  }
#pragma unroll 1
  for (int e = 0; e < 8; ++e) {
    double w = 1.0;
    if (p.kw) w = p.w_f32 ? static_cast<const float*>(p.kw)[d0 + e]
                          : Elem<DT>::to_f32(static_cast<const typename Elem<DT>::T*>(p.kw)[d0 + e]);
    y[e] = f[e] * r * w;
  }
#pragma unroll 1
  for (int e = 0; e < 8; ++e) o[e] = p.inter ? y[e ^ 1] : __shfl_sync(mask, y[e], partner);
  double amax = 0.0;
#pragma unroll 1
  for (int e = 0; e < 8; ++e) {
    const int d = d0 + e;
    if (d < p.rot) {
      const int j = p.inter ? d / 2 : d < half ? d : d - half;
      const bool lead = p.inter ? !(d & 1) : d < half;
      double s, c;
      sincos(pos * static_cast<double>(p.inv_freq[j]), &s, &c);
      y[e] = (lead ? y[e] * c - o[e] * s : y[e] * c + o[e] * s) * static_cast<double>(p.factor);
    }
  }
#pragma unroll 1
  for (int e = 0; e < 8; ++e) amax = fmax(amax, fabs(y[e]));
  amax = fmax(amax, __shfl_xor_sync(mask, amax, 1));
  amax = fmax(amax, __shfl_xor_sync(mask, amax, 2));
  Exact out;
  out.scale = group_scale(static_cast<float>(amax / 7.5));
  const double s = __half2float(out.scale);
  float t[8];
#pragma unroll 1
  for (int e = 0; e < 8; ++e) t[e] = s > 0.0 ? static_cast<float>(fmin(fmax(rint(y[e] / s), -8.0), 7.0)) : 0.0f;
  out.word = pack_codes(t);
  return out;
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 6) append_kernel(const __grid_constant__ AppendParams p) {
  using T16 = typename Elem<DT>::T;
  __shared__ float2 turn[kTok][kD / 2];   // cos, sin
  const int tid = threadIdx.x, lane = tid & 31, sub = tid >> 4, l = lane & 15, d0 = 8 * l;
  const unsigned mask = 0xffffu << (lane & 16);
  const int group = static_cast<int>(blockIdx.x % p.groups);
  const int64_t row0 = static_cast<int64_t>(blockIdx.x / p.groups) * kTok;
  const int tok = static_cast<int>(min(row0 + sub, static_cast<int64_t>(p.T) - 1));
  const bool here = row0 + sub < p.T;
  int b = tok;
  int64_t i = 0, n = 1;
  if (p.cu) {
    b = find_seq(p.cu, p.B, tok);
    const int64_t first = b < p.B ? p.cu[b] : 0;
    i = tok - first;
    n = b < p.B ? min(p.cu[b + 1], p.T) - first : 0;
  }
  const bool live = here && i < n;
  const int len = live ? p.lens[b] : 0;
  const int64_t at = static_cast<int64_t>(len) + i;
  bool fits = live && len >= 0 && static_cast<int64_t>(len) + n <= static_cast<int64_t>(p.pg.max_pages) << p.pg.page_log;
  int pid = 0;
  if (fits) {
    pid = p.pg.tables[b * p.pg.tstride + (at >> p.pg.page_log)];
    fits = pid >= 0 && pid < p.pg.n_pages;
  }
  if (live && !fits && l == 0) report_error(p.status, HQ_ERR_INVALID_ARGUMENT);
  const int place = static_cast<int>(at) & (p.pg.page - 1);
  const double pos = static_cast<double>(at + (live && p.pos_offset ? p.pos_offset[b] : 0));
  const int half = p.rot / 2;
  const int r0 = group * p.rows_per_block, r1 = min(p.Hq + 2 * p.Hkv, r0 + p.rows_per_block);
  if (p.rot > 0 && r0 < p.Hq + p.Hkv && live) {
    for (int j = l; j < half; j += 16) {
      const double turns = pos * static_cast<double>(p.inv_freq[j]) * 0.15915494309189535;
      const double f = 2.0 * (turns - rint(turns));  // angle / pi
      const float h = static_cast<float>(f), r = static_cast<float>(f - h) * 3.14159265f;
      float s, c;
      sincospif(h, &s, &c);
      turn[sub][j] = make_float2(__fmaf_rn(-s, r, c) * p.factor, __fmaf_rn(c, r, s) * p.factor);
    }
  }
  __syncwarp();
  const bool turned = d0 < p.rot;
  const bool lead = d0 < half;
  const int partner = (lane & 16) + (p.inter || !turned ? l : lead ? l + half / 8 : l - half / 8);

  // y_e = r (x_e cs_e + o_e sg_e), o the partner: weights and the angle's cos and sin in one factor
  float cs[8], sg[8], wmax = 0.0f;
  auto factors = [&](const void* w) {
    float wt[8];
    wmax = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      wt[e] = 1.0f;
      if (w) wt[e] = p.w_f32 ? static_cast<const float*>(w)[d0 + e] : Elem<DT>::to_f32(static_cast<const T16*>(w)[d0 + e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float wo = p.inter ? wt[e ^ 1] : __shfl_sync(0xffffffffu, wt[e], partner);
      wmax = fmaxf(wmax, fmaxf(fabsf(wt[e]), fabsf(wo)));
      cs[e] = wt[e];
      sg[e] = 0.0f;
      if (turned && live) {
        const int j = p.inter ? (d0 + e) / 2 : lead ? d0 + e : d0 + e - half;
        const float2 t = turn[sub][j];
        cs[e] = t.x * wt[e];
        sg[e] = ((p.inter ? !(e & 1) : lead) ? -t.y : t.y) * wo;
      }
    }
  };
  auto each = [&](const void* src, const int64_t (&st)[2], int h0, int h1, auto&& row_of) {
    const char* base = static_cast<const char*>(src) + 2 * (tok * st[0] + d0);
    const int64_t step = 2 * st[1];
    uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0;
    if (h0 < h1) x0 = ld_stream(base + h0 * step);
    if (h0 + 1 < h1) x1 = ld_stream(base + (h0 + 1) * step);
#pragma unroll 1
    for (int h = h0; h < h1; ++h) {
      const uint4 x = x0;
      x0 = x1;
      if (h + 2 < h1) x1 = ld_stream(base + (h + 2) * step);
      row_of(h, x);
    }
  };
  auto norm_of = [&](const float (&f)[8]) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __fmaf_rn(f[e], f[e], s);
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    return rsqrtf(__fmaf_rn(s, 1.0f / kD, p.eps));
  };
  auto partners = [&](const uint4& x, const float (&f)[8], float (&o)[8]) {
    if (p.inter) {
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = f[e ^ 1];
    } else {
      uint4 w;
      w.x = __shfl_sync(0xffffffffu, x.x, partner);
      w.y = __shfl_sync(0xffffffffu, x.y, partner);
      w.z = __shfl_sync(0xffffffffu, x.z, partner);
      w.w = __shfl_sync(0xffffffffu, x.w, partner);
      Vec16<DT>::unpack(w, o);
    }
  };
  auto row_ptr = [&](void* base, const int64_t (&st)[2], int h) {
    return reinterpret_cast<uint4*>(static_cast<char*>(base) + 2 * (tok * st[0] + h * st[1] + d0));
  };
  auto put = [&](uint8_t* codes, __half* scales, int h, uint32_t word, __half sc) {
    if (!fits) return;
    uint8_t* row = codes + pid * p.pg.cp + h * p.pg.ch + place * kRowB;
    *reinterpret_cast<uint32_t*>(row + word_at(place, l >> 2, l & 3)) = word;
    if ((l & 3) == 0) scales[pid * p.pg.sp + h * p.pg.sh + place * 4 + (l >> 2)] = sc;
  };

  if (r0 < p.Hq) factors(p.qw);
  each(p.q, p.qs, r0, min(r1, p.Hq), [&](int h, const uint4& x) {
    float f[8], o[8];
    Vec16<DT>::unpack(x, f);
    partners(x, f, o);
    const float r = p.qw ? norm_of(f) : 1.0f;
    uint4 w = x;
    if (live) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = r * __fmaf_rn(f[e], cs[e], o[e] * sg[e]);
      w = make_uint4(pack16<DT>(y[0], y[1]), pack16<DT>(y[2], y[3]), pack16<DT>(y[4], y[5]), pack16<DT>(y[6], y[7]));
    }
    if (live || (here && p.copy_rest)) *row_ptr(p.q_out, p.qos, h) = w;
  });
  const bool plain_k = !p.kw && p.rot == 0;  // k is coded as it came: no rounding before the codes
  if (r1 > p.Hq && r0 < p.Hq + p.Hkv) factors(p.kw);
  each(p.k, p.ks, max(r0 - p.Hq, 0), min(r1 - p.Hq, p.Hkv), [&](int h, const uint4& x) {
    float f[8], o[8], y[8], t[8];
    Vec16<DT>::unpack(x, f);
    partners(x, f, o);
    const float r = p.kw ? norm_of(f) : 1.0f;
    float a = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = r * __fmaf_rn(f[e], cs[e], o[e] * sg[e]);
      a = max_nan(a, fabsf(y[e]));
    }
    a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 1));
    a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 2));
    const float a75 = __fdiv_rn(a, 7.5f);
    __half sc = group_scale(a75);
    const float s = __half2float(sc);
    const float rs = s > 0.0f ? __frcp_rn(s) : 0.0f;
    bool near = false;
    if (!plain_k) {
      // the largest |x w| + |o w_o| of the group at most, for the errors of all its channels
      float size = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) size = fmaxf(size, fabsf(f[e]) + fabsf(o[e]));
      size *= wmax;
      size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, 1));
      size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, 2));
      const float err = size * r * p.slack, e75 = err * 0.13333334f + a75 * 6.0e-8f;
      // the scale's neighbours in float16 are the same for all a it may come from
      near = a75 < INFINITY && __half_as_ushort(group_scale(a75 + e75)) != __half_as_ushort(group_scale(fmaxf(a75 - e75, 0.0f)));
      const float et = __fmaf_rn(err, rs, 2.5e-6f);  // (8 * 2^-22 of the quotient's own roundings)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        t[e] = y[e] * rs;
        const float d = fabsf(t[e] - rintf(t[e]));
        near |= d + et > 0.5f && fabsf(t[e]) < 8.6f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float q0 = y[e] * rs;
        t[e] = __fmaf_rn(__fmaf_rn(-q0, s, y[e]), rs, q0);
      }
    }
    uint32_t word = pack_codes(t);
    if (live) {
      if (__any_sync(mask, near)) {
        const Exact ex = exact_row<DT>(p, x, mask, partner, pos, l);
        word = ex.word;
        sc = ex.scale;
      }
      put(p.pg.k, p.pg.ksc, h, word, sc);
      if (p.k_out)
        *row_ptr(p.k_out, p.kos, h) = make_uint4(pack16<DT>(y[0], y[1]), pack16<DT>(y[2], y[3]),
                                                 pack16<DT>(y[4], y[5]), pack16<DT>(y[6], y[7]));
    }
  });
  each(p.v, p.vs, max(r0 - p.Hq - p.Hkv, 0), r1 - p.Hq - p.Hkv, [&](int h, const uint4& x) {
    float f[8], t[8];
    Vec16<DT>::unpack(x, f);
    float a = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = max_nan(a, fabsf(f[e]));
    a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 1));
    a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 2));
    const __half sc = group_scale(__fdiv_rn(a, 7.5f));
    const float s = __half2float(sc), rs = s > 0.0f ? __frcp_rn(s) : 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q0 = f[e] * rs;
      t[e] = __fmaf_rn(__fmaf_rn(-q0, s, f[e]), rs, q0);
    }
    put(p.pg.v, p.pg.vsc, h, pack_codes(t), sc);
  });
}

template <int DT>
int launch_append(AppendParams p, cudaStream_t st) {
  const int rows = p.Hq + 2 * p.Hkv;
  const int64_t blocks = (static_cast<int64_t>(p.T) + kTok - 1) / kTok;
  // a token's rows stay together (its cos and sin made once) as long as that leaves 4 blocks of 4
  // warps an SM; below, they are split, down to one row each
  const int64_t want = std::max<int64_t>(1, 4LL * current_sm_count() / blocks);
  const int groups = static_cast<int>(std::min<int64_t>(rows, want));
  p.rows_per_block = (rows + groups - 1) / groups;
  p.groups = (rows + p.rows_per_block - 1) / p.rows_per_block;
  if (blocks * p.groups > 0x7fffffff) return HQ_ERR_UNSUPPORTED;
  append_kernel<DT><<<static_cast<unsigned>(blocks * p.groups), kThreads, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HQ_OK : static_cast<int>(e);
}

}  // namespace p4
}  // namespace hq

using namespace hq;

extern "C" int hq_paged4_append(const void* q, const void* k_new, const void* v_new, int x_dtype,
                                const int64_t q_strides[2], const int64_t k_strides[2],
                                const int64_t v_strides[2], int T, int B, int Hq, int Hkv, int D,
                                const int* cu_seqlens, const int* lens, const int* pos_offset,
                                const void* q_weight, const void* k_weight, int w_dtype, float eps,
                                const float* inv_freq, int rotary_dim, int interleaved, float factor,
                                uint8_t* k_codes, uint8_t* v_codes, const int64_t code_strides[2],
                                void* k_scale, void* v_scale, const int64_t scale_strides[2],
                                int n_pages, int page_size, const int* tables, int64_t table_stride,
                                int max_pages, void* q_out, const int64_t qo_strides[2], void* k_out,
                                const int64_t ko_strides[2], int copy_rest, int* status,
                                hq_stream_t stream) {
  if (T < 0 || B < 0 || Hq <= 0 || Hkv <= 0 || rotary_dim < 0 || rotary_dim > D || (rotary_dim > 0 && !inv_freq) ||
      !q_strides || !k_strides || !v_strides || !qo_strides || (k_out && !ko_strides) || !(eps >= 0.0f) ||
      (!cu_seqlens && T != B))
    return HQ_ERR_INVALID_ARGUMENT;
  if (D != p4::kD || rotary_dim % 16 || (x_dtype != HQ_DTYPE_BF16 && x_dtype != HQ_DTYPE_F16) ||
      (w_dtype != x_dtype && w_dtype != HQ_DTYPE_F32) || static_cast<int64_t>(Hq) + 2 * static_cast<int64_t>(Hkv) > 65535)
    return HQ_ERR_UNSUPPORTED;
  const int rc = p4::check_pages(k_codes, v_codes, k_scale, v_scale, code_strides, scale_strides, n_pages,
                                 page_size, tables, table_stride, max_pages, B, Hkv);
  if (rc != HQ_OK) return rc;
  if (T == 0 || B == 0) return T == 0 || !copy_rest ? HQ_OK : HQ_ERR_INVALID_ARGUMENT;
  if (!q || !k_new || !v_new || !q_out || !lens) return HQ_ERR_INVALID_ARGUMENT;
  auto al = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
  if (!al(q) || !al(k_new) || !al(v_new) || !al(q_out) || !al(k_out)) return HQ_ERR_INVALID_ARGUMENT;
  const int64_t* all[5] = {q_strides, k_strides, v_strides, qo_strides, k_out ? ko_strides : qo_strides};
  for (const int64_t* s : all)
    if (s[0] % 8 || s[1] % 8) return HQ_ERR_INVALID_ARGUMENT;
  // what is written has rows of its own
  const int heads[2] = {Hq, Hkv};
  for (int i = 0; i < (k_out ? 2 : 1); ++i)
    if ((T > 1 && all[3 + i][0] == 0) || (heads[i] > 1 && all[3 + i][1] == 0)) return HQ_ERR_INVALID_ARGUMENT;
  p4::AppendParams p{};
  p.pg = p4::make_pages(k_codes, v_codes, k_scale, v_scale, code_strides, scale_strides, n_pages, page_size,
                        tables, table_stride, max_pages);
  p.q = q;
  p.k = k_new;
  p.v = v_new;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = q_strides[i];
    p.ks[i] = k_strides[i];
    p.vs[i] = v_strides[i];
    p.qos[i] = qo_strides[i];
    p.kos[i] = k_out ? ko_strides[i] : 0;
  }
  p.T = T;
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.cu = cu_seqlens;
  p.lens = lens;
  p.pos_offset = pos_offset;
  p.qw = q_weight;
  p.kw = k_weight;
  p.w_f32 = w_dtype == HQ_DTYPE_F32;
  p.eps = eps;
  p.inv_freq = inv_freq;
  p.rot = rotary_dim;
  p.inter = interleaved;
  p.factor = factor;
  p.q_out = q_out;
  p.k_out = k_out;
  p.copy_rest = copy_rest;
  p.status = status;
  p.slack = p4::kSlack * fmaxf(1.0f, fabsf(factor));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return x_dtype == HQ_DTYPE_BF16 ? p4::launch_append<HQ_DTYPE_BF16>(p, st) : p4::launch_append<HQ_DTYPE_F16>(p, st);
}
