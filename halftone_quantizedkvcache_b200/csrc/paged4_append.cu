// New tokens into a paged 4-bit cache, with the norms of q and k per head and the rotation by
// position on the way, in one launch (sm_100a).
//
// Tokens come packed: token r of cu[b] .. cu[b + 1] - 1 is new token i = r - cu[b] of sequence b, at
// cache place lens[b] + i and position P = lens[b] + i + pos_offset[b].  Per row of 128 channels:
// x <- w x / sqrt(mean(x^2) + eps) (with weights), then the first `rot` channels are turned pairwise
// by P * inv_freq[j] (pairs (j, j + rot / 2), or (2j, 2j + 1) interleaved).  q' and k' are rounded
// once, to the model's type; K's codes are those of the unrounded k (paged4.cuh).
//
// Codes are those that float64 arithmetic finds.  P * inv_freq, its cos and its sin are formed in float64
// (once a token, kept as two float32 parts in shared memory); norms and turns are float32, off by at most
// kSlack of the pair's larger value.  The k rows with a quotient or a scale closer to a rounding border than
// that (one in 60) are listed, and formed again in float64 at the end of the block, a warp a row (8 of the
// 126 us below; a half-warp a row 15, on the spot one by one 30).  So are rows of q and k whose squares float32
// does not hold (finding them takes 2 us: their bits are gathered, since a branch in q's loop took 5).  V's codes
// come from its 16-bit values: an 11-bit x over an 11-bit s is 2^-13 away from a border unless it lies on
// it, and one corrected division finds both cases.
//
// Per token (Hq + 2 Hkv) rows are read, Hq (+ Hkv) rows and Hkv 144 bytes written.  16 lanes hold a row
// (8 channels, 16 bytes, each); a half-warp takes one token and all of its rows, 7 of them in flight
// through shared memory (the next row in registers instead: 179 us).
//
// 8 x 4096 tokens of 16 q heads and 8 kv heads, both norms, full rotation, k kept: 126 us, 4.0 TB/s of
// bytes moved.  Bound by issue slots (72 % of them taken; arithmetic units 45 %, DRAM 36 % at half that
// size): for a lane and row of k a reduction of 128 squares, the turn and the codes.  (8 lanes a row, both
// values of a pair in one lane, take 27 % fewer instructions but 96 registers: 131 us, the 20 warps an SM hide
// less.)
#include <algorithm>

#include "paged4.cuh"

namespace hq {
int current_sm_count();

namespace p4 {

constexpr int kThreads = 128;
constexpr int kTok = kThreads / 16;       // tokens per block
constexpr int kRing = 8;                  // rows in flight for each, a power of two
constexpr int kMostRows = 512;            // of a token for a block: its list takes 16 KB

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
};

// Error of the float32 route, relative to |x w cos| + |o w_o sin| (times r and the factor), in units of 2^-24:
// half that of the mean (squares are exact but for 2^-150, below 2^-24 of it where it is a normal number; 3
// sums in a lane's half, the halves, 4 rounds, eps: 10) 5 and that of its root's correction 2.5, cos or sin 1,
// their weight 1 and factor 1, the turn's product 1 and sum 1, r's product 1: 13.5.  The sum is at most the
// pair's length, sqrt(2) times the larger of its turned values.
constexpr float kSlack = 1.4143f * 13.5f / 16777216.0f;

constexpr uint32_t kWhole = 0x80000000u;  // a listed row that float64 writes to q_out or k_out too

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
// The scale of a group from amax / 7.5: NaN where amax is no number, the largest float16 above it.
__device__ __forceinline__ __half group_scale(float a75) {
  if (!(a75 < INFINITY)) return __ushort_as_half(0x7fff);
  return __float2half_rn(fminf(a75, 65504.0f));
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rsqrt_ftz(float x) {  // (infinity below the smallest normal number)
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// a / 7.5 of a 16-bit a, correctly rounded: one correction of the product with 2 / 15
__device__ __forceinline__ float over75(float a) {
  const float q = a * 0.13333334f;
  return a < 1e30f ? __fmaf_rn(__fmaf_rn(-q, 7.5f, a), 0.13333334f, q) : q;
}
// Channels in pairs (e, e + 4): 8 codes become a word of nibbles as one whole number per half.
// k: whole numbers.
__device__ __forceinline__ uint32_t pack_codes(const F2 (&k)[4]) {
  F2 c[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float a, b;
    f2_split(k[e], a, b);
    c[e] = f2_make(fminf(fmaxf(a, -8.0f), 7.0f), fminf(fmaxf(b, -8.0f), 7.0f));
  }
  auto same = [](float x) { return f2_make(x, x); };
  // (8 x 0x1111 makes each code + 8; under 1.5 x 2^23 the low 16 bits hold the number)
  const F2 v = f2_fma(c[3], same(4096.0f), f2_fma(c[2], same(256.0f), f2_fma(c[1], same(16.0f), c[0])));
  const F2 w = f2_add(v, same(12582912.0f + 34952.0f));
  return prmt(f2_lo_bits(w), f2_hi_bits(w), 0x5410u);
}
// rint(x / s) of 16-bit x, s, with rs ~ 1 / s: the quotient corrected once, exact where it is a tie
__device__ __forceinline__ void quotients(const F2 (&x)[4], float s, float rs, F2 (&k)[4]) {
  const F2 ns = f2_make(-s, -s), r2 = f2_make(rs, rs), big = f2_make(12582912.0f, 12582912.0f);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const F2 q = f2_mul(x[e], r2);
    k[e] = f2_sub(f2_add(f2_fma(f2_fma(q, ns, x[e]), r2, q), big), big);
  }
}
template <int DT>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
  if constexpr (DT == HQ_DTYPE_BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <int DT>
__device__ __forceinline__ void unpack_pairs(const uint4& w, F2 (&x)[4]) {
  float f[8];
  Vec16<DT>::unpack(w, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = f2_make(f[e], f[e + 4]);
}
__device__ __forceinline__ float absmax(const F2 (&x)[4]) {  // NaN if any is
  float m = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float a, b;
    f2_split(x[e], a, b);
    m = max_nan(m, max_nan(fabsf(a), fabsf(b)));
  }
  return m;
}
template <int DT>
__device__ __forceinline__ uint4 pack_row(const F2 (&y)[4]) {
  float a[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) f2_split(y[e], a[e], a[e + 4]);
  return make_uint4(pack16<DT>(a[0], a[1]), pack16<DT>(a[2], a[3]), pack16<DT>(a[4], a[5]), pack16<DT>(a[6], a[7]));
}

// The chunk of 8 channels that chunk c is turned with (itself: interleaved pairs, or not turned).
__device__ __forceinline__ int partner_of(const AppendParams& p, int c) {
  const int h8 = p.rot / 16;
  return p.inter || c >= 2 * h8 ? c : c < h8 ? c + h8 : c - h8;
}
template <int DT>
__device__ __forceinline__ float weight_at(const AppendParams& p, const void* w, int d) {
  if (!w) return 1.0f;
  return p.w_f32 ? static_cast<const float*>(w)[d] : Elem<DT>::to_f32(static_cast<const typename Elem<DT>::T*>(w)[d]);
}

// A row of q or k in float64 (a warp, 4 channels a lane): `out` takes it and `codes` and `scales` its codes, where
// they are not null.
template <int DT>
__device__ __forceinline__ void exact_row(const AppendParams& p, const void* weights, const char* row, const float4* turn,
                                          char* out, uint8_t* codes, __half* scales, int place) {
  const int lane = threadIdx.x & 31, c = lane >> 1, half = p.rot / 2;
  const int d0 = 4 * lane, o0 = 8 * partner_of(p, c) + 4 * (lane & 1);  // (interleaved: partners e ^ 1)
  auto unpack = [](const uint2& w, float (&f)[4]) {
    const float2 a = unpack16<DT>(w.x), b = unpack16<DT>(w.y);
    f[0] = a.x;
    f[1] = a.y;
    f[2] = b.x;
    f[3] = b.y;
  };
  float f[4], g[4], wt[4], wo[4];
  const uint2 x = *reinterpret_cast<const uint2*>(row + 2 * d0), xo = *reinterpret_cast<const uint2*>(row + 2 * o0);
  float4 t[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int d = d0 + e, eo = p.inter ? e ^ 1 : e;
    wt[e] = weight_at<DT>(p, weights, d);
    wo[e] = weight_at<DT>(p, weights, o0 + eo);
    t[e] = turn[d >= p.rot ? 0 : p.inter ? d / 2 : d < half ? d : d - half];
  }
  unpack(x, f);
  unpack(xo, g);
  double r = 1.0;
  if (weights) {
    double s = fma(static_cast<double>(f[0]), static_cast<double>(f[0]), static_cast<double>(f[1]) * f[1]) +
               fma(static_cast<double>(f[2]), static_cast<double>(f[2]), static_cast<double>(f[3]) * f[3]);
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    s = s * (1.0 / kD) + static_cast<double>(p.eps);
    // (times 2^-200 or 2^200 where float32 would not hold it, its root by 2^-100 or 2^100)
    const double by = s > 1e36 ? 0x1p-100 : s < 1e-30 ? 0x1p100 : 1.0;
    s *= by * by;
    r = rsqrtf(static_cast<float>(s));
    r = r * fma(-0.5 * s * r, r, 1.5) * by;  // 2^-22 becomes 2^-43
  }
  double z[4], amax = 0.0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    z[e] = f[e] * r * static_cast<double>(wt[e]);
    if (d0 < p.rot) {
      const double o = (p.inter ? g[e ^ 1] : g[e]) * r * static_cast<double>(wo[e]);
      const double cs = static_cast<double>(t[e].x) + t[e].z, sn = static_cast<double>(t[e].y) + t[e].w;
      z[e] = ((p.inter ? !(e & 1) : d0 < half) ? z[e] * cs - o * sn : z[e] * cs + o * sn) * static_cast<double>(p.factor);
    }
    if (fabs(z[e]) > amax || z[e] != z[e]) amax = fabs(z[e]);  // (NaN if any is: nothing is above it)
  }
  __syncwarp();                           // (the row has been read, by all lanes: out may be its memory)
  if (out)
    *reinterpret_cast<uint2*>(out + 2 * d0) = make_uint2(pack16<DT>(static_cast<float>(z[0]), static_cast<float>(z[1])),
                                                         pack16<DT>(static_cast<float>(z[2]), static_cast<float>(z[3])));
  if (!codes) return;                     // (the same for all lanes)
  float a75 = static_cast<float>(amax * (2.0 / 15.0));
#pragma unroll
  for (int m = 4; m >= 1; m >>= 1) a75 = max_nan(a75, __shfl_xor_sync(0xffffffffu, a75, m));
  const __half sc = group_scale(a75);
  const float s = __half2float(sc);
  double rs = 0.0;
  if (s > 0.0f) {
    rs = rcp(s);
    rs = rs * fma(-static_cast<double>(s), rs, 2.0);
  }
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {           // (channels that are not turned can lie on a border: corrected, exact there)
    const double q = z[e] * rs;
    const float k = static_cast<float>(rint(fma(fma(-q, static_cast<double>(s), z[e]), rs, q)));
    word |= static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(k, -8.0f), 7.0f)) + 8) << (4 * e);
  }
  const int g4 = lane >> 3, j = c & 3;
  *reinterpret_cast<uint16_t*>(codes + word_at(place, g4, j) + 2 * (lane & 1)) = static_cast<uint16_t>(word);
  if ((lane & 7) == 0) scales[g4] = sc;
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 7) append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ uint4 ring[kTok][kRing * 16];
  __shared__ float4 turn[kTok][kD / 2];   // cos and sin, and what is left of them
  extern __shared__ uint32_t again[];     // rows to form again: kWhole or 0, token of the block, row
  __shared__ int n_again;
  __shared__ int4 where[kTok];
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
  const bool live = here && i >= 0 && i < n;
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
  const bool plain_k = !p.kw && p.rot == 0;  // k is coded as it came: no rounding before the codes
  if (l == 0) where[sub] = make_int4(tok, pid, place, fits);
  if (tid == 0) n_again = 0;
  __syncthreads();
  const int half = p.rot / 2;
  const int r0 = group * p.rows_per_block, r1 = min(p.Hq + 2 * p.Hkv, r0 + p.rows_per_block);
  // rows r0 .. r1 - 1 (q heads, k heads, v heads) arrive in order through a ring of this half-warp's; a
  // lane copies and reads its own 16 bytes
  const uint4* slots = ring[sub] + l;
  const uint32_t slots_at = smem_u32(slots);
  int ahead = r0, turn_at = 0;            // the next row to fetch, the first of another tensor
  const char* from = nullptr;
  int64_t step = 0;
  auto fetch = [&]() {
    if (ahead >= turn_at && ahead < r1) {
      const int h0 = ahead < p.Hq ? 0 : ahead < p.Hq + p.Hkv ? p.Hq : p.Hq + p.Hkv;  // the tensor's first row
      const void* base = ahead < p.Hq ? p.q : ahead < p.Hq + p.Hkv ? p.k : p.v;
      const int64_t* st = ahead < p.Hq ? p.qs : ahead < p.Hq + p.Hkv ? p.ks : p.vs;
      from = static_cast<const char*>(base) + 2 * (tok * st[0] + (ahead - h0) * st[1] + d0);
      step = 2 * st[1];
      turn_at = ahead < p.Hq ? p.Hq : ahead < p.Hq + p.Hkv ? p.Hq + p.Hkv : 0x7fffffff;
    }
    if (ahead < r1)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slots_at + 256 * (ahead & (kRing - 1))), "l"(from) : "memory");
    cp_async_commit();                    // (a group a row, there or not)
    from += step;
    ++ahead;
  };
#pragma unroll 1
  for (int i = 0; i < kRing - 1; ++i) fetch();
  if (p.rot > 0 && r0 < p.Hq + p.Hkv && live) {
#pragma unroll 2
    for (int j = l; j < half; j += 16) {
      const double turns = pos * static_cast<double>(p.inv_freq[j]) * 0.15915494309189535;
      double s, c;
      sincospi(2.0 * (turns - rint(turns)), &s, &c);
      const float ch = static_cast<float>(c), sh = static_cast<float>(s);
      turn[sub][j] = make_float4(ch, sh, static_cast<float>(c - ch), static_cast<float>(s - sh));
    }
  }
  __syncwarp();
  const bool turned = d0 < p.rot;
  const bool lead = d0 < half;
  const int partner = (lane & 16) + (p.inter || !turned ? l : lead ? l + half / 8 : l - half / 8);

  // y = r (x cs + o sg), o the partner: weights, factor and the angle's cos and sin in one
  F2 cs[4], sg[4];
  auto factors = [&](const void* w) {
    float wt[8], c[8], g[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      wt[e] = weight_at<DT>(p, w, d0 + e);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float wo = p.inter ? wt[e ^ 1] : __shfl_sync(0xffffffffu, wt[e], partner);
      c[e] = wt[e];
      g[e] = 0.0f;
      if (turned && live) {
        const int j = p.inter ? (d0 + e) / 2 : lead ? d0 + e : d0 + e - half;
        const float2 t = *reinterpret_cast<const float2*>(&turn[sub][j]);
        c[e] = t.x * (wt[e] * p.factor);
        g[e] = ((p.inter ? !(e & 1) : lead) ? -t.y : t.y) * (wo * p.factor);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      cs[e] = f2_make(c[e], c[e + 4]);
      sg[e] = f2_make(g[e], g[e + 4]);
    }
  };
  auto each = [&](int from, int to, auto&& row_of) {
#pragma unroll 1
    for (int r = from; r < to; ++r) {
      cp_async_wait<kRing - 2>();
      const uint4 x = slots[16 * (r & (kRing - 1))];
      fetch();                            // where the row before was
      row_of(x);
    }
  };
  auto mean_square = [&](const F2 (&f)[4]) {
    F2 s2 = f2_mul(f[0], f[0]);
#pragma unroll
    for (int e = 1; e < 4; ++e) s2 = f2_fma(f[e], f[e], s2);
    float s, s1;
    f2_split(s2, s, s1);
    s += s1;
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    return __fmaf_rn(s, 1.0f / kD, p.eps);
  };
  // Normed and turned row; whether float32 holds its norm: bf16's largest and smallest rows have a mean square that
  // is infinite or no normal number in float32.  Their 1 / root is then infinite or NaN, and so is all of the row.
  auto turned_row = [&](const uint4& x, bool norm, F2 (&y)[4]) {
    F2 f[4], o[4];
    unpack_pairs<DT>(x, f);
    if (p.inter) {                        // partners e ^ 1: the halves of the words
      unpack_pairs<DT>(make_uint4(prmt(x.x, 0, 0x1032u), prmt(x.y, 0, 0x1032u), prmt(x.z, 0, 0x1032u), prmt(x.w, 0, 0x1032u)), o);
    } else {
      uint4 w;
      w.x = __shfl_sync(0xffffffffu, x.x, partner);
      w.y = __shfl_sync(0xffffffffu, x.y, partner);
      w.z = __shfl_sync(0xffffffffu, x.z, partner);
      w.w = __shfl_sync(0xffffffffu, x.w, partner);
      unpack_pairs<DT>(w, o);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = f2_fma(f[e], cs[e], f2_mul(o[e], sg[e]));
    if (!norm) return true;
    const float s = mean_square(f);
    float r = rsqrt_ftz(s);
    r *= __fmaf_rn(-0.5f * s * r, r, 1.5f);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = f2_mul(y[e], f2_make(r, r));
    return fabsf(r) < INFINITY;
  };
  auto list = [&](int row, uint32_t whole) { again[atomicAdd(&n_again, 1)] = whole | static_cast<uint32_t>(sub << 16 | row); };

  if (r0 < p.Hq) {
    factors(p.qw);
    char* to = static_cast<char*>(p.q_out) + 2 * (tok * p.qos[0] + r0 * p.qos[1] + d0);
    const bool store = live || (here && p.copy_rest);
#pragma unroll 1
    for (int c = r0; c < min(r1, p.Hq); c += 32) {
      const int end = min(c + 32, min(r1, p.Hq));
      uint32_t odd = 0;                   // the rows for float64, the last in bit 0
      each(c, end, [&](const uint4& x) {
        F2 y[4];
        const bool held = turned_row(x, p.qw, y);
        const uint4 w = live ? pack_row<DT>(y) : x;
        if (store && (held || !live)) *reinterpret_cast<uint4*>(to) = w;  // (others stay what they were: q_out may be q)
        odd = 2 * odd + !held;
        to += 2 * p.qos[1];
      });
      if (live && l == 0)
        for (; odd; odd &= odd - 1) list(end - __ffs(odd), kWhole);
    }
  }
  // a lane's word and its group's scale in a head's page
  const int64_t code_at = pid * p.pg.cp + place * kRowB + word_at(place, l >> 2, l & 3);
  const int64_t scale_at = pid * p.pg.sp + place * 4 + (l >> 2);
  if (r1 > p.Hq && r0 < p.Hq + p.Hkv) {
    factors(p.kw);
    const int h0 = max(r0 - p.Hq, 0);
    uint8_t* codes = p.pg.k + code_at + h0 * p.pg.ch;
    __half* scales = p.pg.ksc + scale_at + h0 * p.pg.sh;
    char* to = static_cast<char*>(p.k_out) + 2 * (tok * p.kos[0] + h0 * p.kos[1] + d0);
    int h = h0;
    each(p.Hq + h0, min(r1, p.Hq + p.Hkv), [&](const uint4& x) {
      F2 y[4], k[4];
      turned_row(x, p.kw, y);
      float a = absmax(y);
      a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 1));
      a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 2));
      const float a75 = over75(a);
      const __half sc = group_scale(a75);
      const float s = __half2float(sc), rs = s > 0.0f ? rcp(s) : 0.0f;
      bool near = false;
      if (!plain_k) {
        const float err = kSlack * fmaxf(a, p.inter ? a : __shfl_sync(0xffffffffu, a, partner));
        const float e75 = __fmaf_rn(err, 0.13333334f, a75 * 1.2e-7f);
        // the scale is the same for all a75 that this one may stand for; or the row's norm is for float64 (or it
        // holds no numbers)
        near = !(a75 < INFINITY) || __half_as_ushort(group_scale(a75 + e75)) != __half_as_ushort(group_scale(fmaxf(a75 - e75, 0.0f)));
        const F2 r2 = f2_make(rs, rs), big = f2_make(12582912.0f, 12582912.0f);  // 1.5 x 2^23
        float far = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const F2 t = f2_mul(y[e], r2);
          k[e] = f2_sub(f2_add(t, big), big);
          float d0, d1;
          f2_split(f2_sub(t, k[e]), d0, d1);
          far = fmaxf(far, fmaxf(fabsf(d0), fabsf(d1)));
        }
        near |= far + __fmaf_rn(err, rs, 4e-6f) > 0.5f;  // (8 x 2^-21 of the quotient's own roundings)
      } else {
        quotients(y, s, rs, k);
      }
      const uint32_t word = pack_codes(k);
      if (live) {
        if (__any_sync(mask, near) && l == 0) list(p.Hq + h, a75 < INFINITY ? 0 : kWhole);
        if (fits) {
          *reinterpret_cast<uint32_t*>(codes) = word;
          if ((l & 3) == 0) *scales = sc;
        }
        if (p.k_out) *reinterpret_cast<uint4*>(to) = pack_row<DT>(y);
      }
      codes += p.pg.ch;
      scales += p.pg.sh;
      to += 2 * p.kos[1];
      ++h;
    });
  }
  if (r1 > p.Hq + p.Hkv) {
    const int h0 = max(r0 - p.Hq - p.Hkv, 0);
    uint8_t* codes = p.pg.v + code_at + h0 * p.pg.ch;
    __half* scales = p.pg.vsc + scale_at + h0 * p.pg.sh;
    each(p.Hq + p.Hkv + h0, r1, [&](const uint4& x) {
      F2 f[4], k[4];
      unpack_pairs<DT>(x, f);
      float a = absmax(f);
      a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 1));
      a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 2));
      const __half sc = group_scale(over75(a));
      const float s = __half2float(sc);
      quotients(f, s, s > 0.0f ? rcp(s) : 0.0f, k);
      const uint32_t word = pack_codes(k);
      if (fits) {
        *reinterpret_cast<uint32_t*>(codes) = word;
        if ((l & 3) == 0) *scales = sc;
      }
      codes += p.pg.ch;
      scales += p.pg.sh;
    });
  }
  // ---- rows whose norm float32 does not hold, or whose codes it could not tell
  const bool lists = (r0 < p.Hq && p.qw) || (r1 > p.Hq && r0 < p.Hq + p.Hkv && !plain_k);
  if (!lists) return;
  __syncthreads();
  for (int i = tid >> 5; i < n_again; i += kThreads / 32) {
    const uint32_t entry = again[i];
    const int of = entry >> 16 & 0xff, row = entry & 0xffff, h = row - p.Hq;
    const int4 w = where[of];             // token, page, place, whether it has one
    const bool of_q = row < p.Hq;
    const int64_t* from = of_q ? p.qs : p.ks;
    const int64_t* to = of_q ? p.qos : p.kos;
    const int head = of_q ? row : h;
    char* out = static_cast<char*>(of_q ? p.q_out : p.k_out);
    exact_row<DT>(p, of_q ? p.qw : p.kw, static_cast<const char*>(of_q ? p.q : p.k) + 2 * (w.x * from[0] + head * from[1]), turn[of],
                  out && entry & kWhole ? out + 2 * (w.x * to[0] + head * to[1]) : nullptr,
                  !of_q && w.w ? p.pg.k + w.y * p.pg.cp + h * p.pg.ch + w.z * kRowB : nullptr,
                  p.pg.ksc + w.y * p.pg.sp + h * p.pg.sh + w.z * 4, w.z);
  }
}

template <int DT>
int launch_append(AppendParams p, cudaStream_t st) {
  const int rows = p.Hq + 2 * p.Hkv;
  const int64_t blocks = (static_cast<int64_t>(p.T) + kTok - 1) / kTok;
  // a token's rows stay together (its cos and sin made once) as long as that leaves 8 blocks of 4
  // warps an SM; below, they are split, down to one row each
  const int64_t want = std::max<int64_t>(1, 8LL * current_sm_count() / blocks);
  const int groups = static_cast<int>(std::min<int64_t>(rows, want));
  p.rows_per_block = std::min((rows + groups - 1) / groups, kMostRows);
  p.groups = (rows + p.rows_per_block - 1) / p.rows_per_block;
  if (blocks * p.groups > 0x7fffffff) return HQ_ERR_UNSUPPORTED;
  const int list = kTok * std::min(p.rows_per_block, p.Hq + p.Hkv) * 4;  // a block's q and k rows
  append_kernel<DT><<<static_cast<unsigned>(blocks * p.groups), kThreads, list, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HQ_OK : static_cast<int>(e);
}

}  // namespace p4
}  // namespace hq

using namespace hq;

extern "C" int hq_paged4_append(const hq_paged4_append_args* args) {
  if (!args) return HQ_ERR_INVALID_ARGUMENT;
  const hq_paged4_append_args& a = *args;
  if (a.T < 0 || a.B < 0 || a.Hq <= 0 || a.Hkv <= 0 || a.rotary_dim < 0 || a.rotary_dim > a.D ||
      (a.rotary_dim > 0 && !a.inv_freq) || !(a.eps >= 0.0f) || (!a.cu_seqlens && a.T != a.B))
    return HQ_ERR_INVALID_ARGUMENT;
  if (a.D != p4::kD || a.rotary_dim % 16 || (a.x_dtype != HQ_DTYPE_BF16 && a.x_dtype != HQ_DTYPE_F16) ||
      (a.w_dtype != a.x_dtype && a.w_dtype != HQ_DTYPE_F32) || static_cast<int64_t>(a.Hq) + 2 * static_cast<int64_t>(a.Hkv) > 65535)
    return HQ_ERR_UNSUPPORTED;
  const int rc = p4::check_pages(a.k_codes, a.v_codes, a.k_scale, a.v_scale, a.code_strides, a.scale_strides, a.n_pages,
                                 a.page_size, a.tables, a.table_stride, a.max_pages, a.B, a.Hkv);
  if (rc != HQ_OK) return rc;
  if (a.T == 0 || a.B == 0) return a.T == 0 || !a.copy_rest ? HQ_OK : HQ_ERR_INVALID_ARGUMENT;
  if (!a.q || !a.k_new || !a.v_new || !a.q_out || !a.lens) return HQ_ERR_INVALID_ARGUMENT;
  auto al = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
  if (!al(a.q) || !al(a.k_new) || !al(a.v_new) || !al(a.q_out) || !al(a.k_out)) return HQ_ERR_INVALID_ARGUMENT;
  const int64_t* all[5] = {a.q_strides, a.k_strides, a.v_strides, a.qo_strides, a.k_out ? a.ko_strides : a.qo_strides};
  for (const int64_t* s : all)
    if (s[0] % 8 || s[1] % 8) return HQ_ERR_INVALID_ARGUMENT;
  // What is written has memory of its own, apart from the inputs', which other blocks may still read and this one
  // reads a second time; but q_out may be q, whose rows one block reads and writes.
  const Rows q = packed_rows(a.q, a.T, a.Hq, a.q_strides), k = packed_rows(a.k_new, a.T, a.Hkv, a.k_strides),
             v = packed_rows(a.v_new, a.T, a.Hkv, a.v_strides), qo = packed_rows(a.q_out, a.T, a.Hq, a.qo_strides);
  if (rows_meet(qo) || (!same_rows(qo, q) && rows_meet(qo, q)) || rows_meet(qo, k) || rows_meet(qo, v))
    return HQ_ERR_INVALID_ARGUMENT;
  if (a.k_out) {
    const Rows ko = packed_rows(a.k_out, a.T, a.Hkv, a.ko_strides);
    if (rows_meet(ko) || rows_meet(ko, q) || rows_meet(ko, k) || rows_meet(ko, v) || rows_meet(ko, qo)) return HQ_ERR_INVALID_ARGUMENT;
  }
  if (!p4::own_memory(a.k_codes, a.v_codes, a.code_strides, 1, p4::kRowB, a.n_pages, a.Hkv, a.page_size) ||
      !p4::own_memory(a.k_scale, a.v_scale, a.scale_strides, 2, p4::kScaleB, a.n_pages, a.Hkv, a.page_size))
    return HQ_ERR_INVALID_ARGUMENT;
  p4::AppendParams p{};
  p.pg = p4::make_pages(a.k_codes, a.v_codes, a.k_scale, a.v_scale, a.code_strides, a.scale_strides, a.n_pages, a.page_size,
                        a.tables, a.table_stride, a.max_pages);
  p.q = a.q;
  p.k = a.k_new;
  p.v = a.v_new;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = a.q_strides[i];
    p.ks[i] = a.k_strides[i];
    p.vs[i] = a.v_strides[i];
    p.qos[i] = a.qo_strides[i];
    p.kos[i] = a.k_out ? a.ko_strides[i] : 0;
  }
  p.T = a.T;
  p.B = a.B;
  p.Hq = a.Hq;
  p.Hkv = a.Hkv;
  p.cu = a.cu_seqlens;
  p.lens = a.lens;
  p.pos_offset = a.pos_offset;
  p.qw = a.q_weight;
  p.kw = a.k_weight;
  p.w_f32 = a.w_dtype == HQ_DTYPE_F32;
  p.eps = a.eps;
  p.inv_freq = a.inv_freq;
  p.rot = a.rotary_dim;
  p.inter = a.interleaved;
  p.factor = a.factor;
  p.q_out = a.q_out;
  p.k_out = a.k_out;
  p.copy_rest = a.copy_rest;
  p.status = a.status;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a.stream);
  return a.x_dtype == HQ_DTYPE_BF16 ? p4::launch_append<HQ_DTYPE_BF16>(p, st) : p4::launch_append<HQ_DTYPE_F16>(p, st);
}
