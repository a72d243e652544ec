// Rotary positions and the write of new tokens into an int8 cache, in one launch, for
// batches whose sequences have lengths of their own (sm_100a).
//
// Token i of sequence b has position P = lens[b] + i + pos_offset[b].  The first `rot`
// channels of each q and k row are turned pairwise by P * inv_freq[j] (pairs (j, j + rot/2),
// or (2j, 2j + 1) interleaved): (x, y) -> c (x cos - y sin), c (y cos + x sin), with one
// factor c for scaled positions.  Rotated q goes to q_out; rotated k is coded with the
// cache's own per-channel scale, clamp(rint(k / k_scale), +-127); v with its own per-token
// scale max(amax, 1e-8) / 127, which is stored; both land in cache row lens[b] + i.
//
// Exactness.  P * inv_freq has at most 31 + 24 significant bits and is formed in float64;
// angles near 10^6 rad would be off by 0.06 rad in float32.  k is never rounded to the
// model's type between rotation and coding, and a code is the nearest integer of the
// float64 quotient: one rounding of the exact value.  The 16-bit kernel gets there mostly in
// float32: the angle's fraction of a turn is taken in float64 and kept as a float32 pair, the
// turned values are off by 2^-22 of the pair's size at most, and a quotient closer to a
// rounding border than that (about one in 10^4) is formed again in float64.
//
// A q element is read and written (4 bytes), a k or v element read and coded (3 bytes).  A lane
// holds 8 channels (16 bytes), D / 8 lanes a row, and keeps the cos and sin of its channels for all
// rows of its token.  8 sequences x 4096 tokens, 16 + 8 + 8 heads, bf16: 144 us, 3.3 TB/s of the
// 470 MB it cannot do without (0.50 of measured).  Bound by latency: issue slots are 60 % full and
// memory half, since no load is in flight while a warp forms its sines and two are in between.  The
// kernel for float32 and for rotary sizes off the lanes' grid forms every channel in float64: 402 us
// (2.2 TB/s of 873 MB) and, bf16 with 72 channels turned, 387 us at the same sizes.
#include <algorithm>
#include <cmath>

#include "hq_common.cuh"

namespace hq {
int current_sm_count();

namespace rope {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct Params {
  const void* q;
  const void* k;
  const void* v;
  int64_t qs[3], ks[3], vs[3];   // (b, h, s) element strides
  int Hq, Hkv, S, D;
  const float* inv_freq;
  int rot, inter;
  float factor;
  const int* lens;
  const int* n_new;
  const int* pos_offset;
  const void* ksc;
  int s_dt;
  int64_t kss[3];
  int8_t* kc;
  int8_t* vc;
  int64_t cs[3];
  void* vsc;
  int64_t vss[3];
  int cap;
  void* q_out;
  int64_t qos[3];
  int* status;
  int rows_per_block;
  int64_t tokens;                // 16-bit kernel
  int groups, ks_vec;
  float slack;                   // 2^-21 max(1, |factor|)
};

// CPL consecutive channels of a row
template <int DT, int CPL>
__device__ __forceinline__ void load_n(const void* base, int64_t i, float (&f)[CPL]) {
  using T = typename Elem<DT>::T;
  struct alignas(sizeof(T) * CPL > 16 ? 16 : sizeof(T) * CPL) Pack { T x[CPL]; };
  const Pack pk = *reinterpret_cast<const Pack*>(static_cast<const T*>(base) + i);
#pragma unroll
  for (int e = 0; e < CPL; ++e) f[e] = Elem<DT>::to_f32(pk.x[e]);
}
template <int DT, int CPL>
__device__ __forceinline__ void store_n(void* base, int64_t i, const float (&f)[CPL]) {
  using T = typename Elem<DT>::T;
  struct alignas(sizeof(T) * CPL > 16 ? 16 : sizeof(T) * CPL) Pack { T x[CPL]; };
  Pack pk;
#pragma unroll
  for (int e = 0; e < CPL; ++e) pk.x[e] = Elem<DT>::from_f32(f[e]);
  *reinterpret_cast<Pack*>(static_cast<T*>(base) + i) = pk;
}
template <int CPL>
__device__ __forceinline__ void store_codes(int8_t* dst, const int (&c)[CPL]) {
  struct alignas(CPL) Pack { int8_t x[CPL]; };
  Pack pk;
#pragma unroll
  for (int e = 0; e < CPL; ++e) pk.x[e] = static_cast<int8_t>(c[e]);
  *reinterpret_cast<Pack*>(dst) = pk;
}

// Block (token b * S + i, group of rows): warps take rows of the token's Hq q heads, Hkv k
// heads and Hkv v heads; a lane holds D / 32 channels.
template <int DT, int D>
__global__ void __launch_bounds__(kThreads) rope_append_kernel(const Params p) {
  constexpr int CPL = D / 32;
  using T = typename Elem<DT>::T;
  __shared__ double2 turn[D / 2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / p.S, i = blockIdx.x % p.S;
  const int len = p.lens[b];
  const int n = p.n_new ? min(max(p.n_new[b], 0), p.S) : p.S;
  const bool live = i < n;
  const int64_t row = static_cast<int64_t>(len) + i;
  const bool fits = len >= 0 && static_cast<int64_t>(len) + n <= p.cap;
  if (live && !fits && tid == 0) report_error(p.status, HQ_ERR_INVALID_ARGUMENT);
  if (live) {
    const double pos = static_cast<double>(row + (p.pos_offset ? p.pos_offset[b] : 0));
    for (int j = tid; j < p.rot / 2; j += kThreads) {
      double s, c;
      sincos(pos * static_cast<double>(p.inv_freq[j]), &s, &c);
      turn[j] = make_double2(c * p.factor, s * p.factor);
    }
  }
  __syncthreads();
  const int rows = p.Hq + 2 * p.Hkv;
  const int r_end = min(rows, (static_cast<int>(blockIdx.y) + 1) * p.rows_per_block);
  for (int r = blockIdx.y * p.rows_per_block + warp; r < r_end; r += kWarps) {
    const int d0 = lane * CPL;
    if (r < p.Hq + p.Hkv) {
      const bool is_q = r < p.Hq;
      if (!is_q && !(live && fits)) continue;
      const int h = is_q ? r : r - p.Hq;
      const void* src = is_q ? p.q : p.k;
      const int64_t* st = is_q ? p.qs : p.ks;
      const int64_t base = b * st[0] + h * st[1] + i * st[2];
      float x[CPL];
      load_n<DT, CPL>(src, base + d0, x);
      double y[CPL];
#pragma unroll
      for (int e = 0; e < CPL; ++e) {
        const int d = d0 + e;
        y[e] = x[e];
        if (live && d < p.rot) {
          int j, other;
          bool lead;
          if (p.inter) {
            j = d >> 1;
            lead = !(d & 1);
            other = d ^ 1;
          } else {
            lead = d < p.rot / 2;
            j = lead ? d : d - p.rot / 2;
            other = lead ? d + p.rot / 2 : j;
          }
          const double o = Elem<DT>::to_f32(static_cast<const T*>(src)[base + other]);
          const double2 t = turn[j];
          y[e] = lead ? x[e] * t.x - o * t.y : x[e] * t.x + o * t.y;
        }
      }
      __syncwarp();  // the row is read before any of it is written (q_out may be q)
      if (is_q) {
        float f[CPL];
#pragma unroll
        for (int e = 0; e < CPL; ++e) f[e] = live ? static_cast<float>(y[e]) : x[e];
        store_n<DT, CPL>(p.q_out, b * p.qos[0] + h * p.qos[1] + i * p.qos[2] + d0, f);
      } else {
        int c[CPL];
#pragma unroll
        for (int e = 0; e < CPL; ++e) {
          const int64_t si = b * p.kss[0] + h * p.kss[1] + (d0 + e) * p.kss[2];
          const double s = p.s_dt == HQ_DTYPE_F16 ? __half2float(static_cast<const __half*>(p.ksc)[si])
                                                  : static_cast<const float*>(p.ksc)[si];
          c[e] = static_cast<int>(fmin(fmax(rint(y[e] / s), -127.0), 127.0));
        }
        store_codes<CPL>(p.kc + b * p.cs[0] + h * p.cs[1] + row * p.cs[2] + d0, c);
      }
    } else if (live && fits) {
      const int h = r - p.Hq - p.Hkv;
      float x[CPL];
      load_n<DT, CPL>(p.v, b * p.vs[0] + h * p.vs[1] + i * p.vs[2] + d0, x);
      float m = 0.0f;
#pragma unroll
      for (int e = 0; e < CPL; ++e) m = fmaxf(m, fabsf(x[e]));
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const Quantizer qz = Quantizer::from_amax(m);
      int c[CPL];
#pragma unroll
      for (int e = 0; e < CPL; ++e) c[e] = qz.code(x[e]);
      store_codes<CPL>(p.vc + b * p.cs[0] + h * p.cs[1] + row * p.cs[2] + d0, c);
      if (lane == 0) {
        const int64_t so = b * p.vss[0] + h * p.vss[1] + row * p.vss[2];
        if (p.s_dt == HQ_DTYPE_F16) static_cast<__half*>(p.vsc)[so] = __float2half_rn(qz.scale);
        else static_cast<float*>(p.vsc)[so] = qz.scale;
      }
    }
  }
}

// ---------------------------------------------------------------- 16-bit types
// Code of one k channel in float64: x turned with its partner o by the angle (lead: x is the
// first of the pair; turned: the channel is rotated at all).
__device__ __noinline__ int exact_code(float x, float o, bool lead, bool turned, double angle,
                                       double factor, float scale) {
  double y = x;
  if (turned) {
    double s, c;
    sincos(angle, &s, &c);
    c *= factor;
    s *= factor;
    y = lead ? x * c - o * s : x * c + o * s;
  }
  return static_cast<int>(fmin(fmax(rint(y / scale), -127.0), 127.0));
}
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
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

// D / 8 lanes per token; a warp takes 32 / (D / 8) neighbouring tokens and `rows_per_block`
// rows of each (the same ones, so that its branches agree).  Needs rot % 16 == 0: the partner
// of a lane's 8 channels is another lane's 8 (or, interleaved, the lane's own).
constexpr int kThreads16 = 128;
// resident blocks per SM that the registers are held to: 8 x 4096 tokens took 189 us with none
// (110 registers, 4 blocks), 151 / 141 / 149 / 167 us for 5 / 6 / 8 / 10
constexpr int kBlocks16 = 6;
template <int DT, int D>
__global__ void __launch_bounds__(kThreads16, kBlocks16) rope_append16_kernel(const __grid_constant__ Params p) {
  constexpr int LPR = D / 8, TPW = 32 / LPR;
  using E = Elem<DT>;
  const int lane = threadIdx.x & 31, sub = lane / LPR, l = lane % LPR, d0 = 8 * l;
  const int64_t wg = static_cast<int64_t>(blockIdx.x) * (kThreads16 / 32) + (threadIdx.x >> 5);
  const int rows = p.Hq + 2 * p.Hkv;
  const int64_t first = wg / p.groups * TPW;
  if (first >= p.tokens) return;  // the whole warp
  const bool here = first + sub < p.tokens;
  const int64_t token = here ? first + sub : first;
  const int r0 = static_cast<int>(wg % p.groups) * p.rows_per_block, r1 = min(rows, r0 + p.rows_per_block);
  const int b = static_cast<int>(token / p.S), i = static_cast<int>(token - static_cast<int64_t>(b) * p.S);
  const int len = p.lens[b];
  const int n = p.n_new ? min(max(p.n_new[b], 0), p.S) : p.S;
  const bool live = here && i < n;
  const int64_t row = static_cast<int64_t>(len) + i;
  const bool fits = len >= 0 && static_cast<int64_t>(len) + n <= p.cap;
  if (live && !fits && l == 0) report_error(p.status, HQ_ERR_INVALID_ARGUMENT);
  const bool write = live && fits;
  const double pos = static_cast<double>(row + (p.pos_offset ? p.pos_offset[b] : 0));
  const int half = p.rot / 2;
  const bool turned = d0 < p.rot;
  const bool lead = d0 < half;                 // half layout: this lane's side of its pairs
  const int j0 = p.inter ? d0 / 2 : lead ? d0 : d0 - half;
  // y = x cs + o sg, o the partner
  float cs[8], sg[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.0f;
    sg[e] = 0.0f;
  }
  if (turned && r0 < p.Hq + p.Hkv) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (p.inter && (e & 1)) {
        cs[e] = cs[e - 1];
        sg[e] = -sg[e - 1];
        continue;
      }
      const int j = j0 + (p.inter ? e / 2 : e);
      const double turns = pos * static_cast<double>(p.inv_freq[j]) * 0.15915494309189535;
      const double f = 2.0 * (turns - rint(turns));  // angle / pi
      const float h = static_cast<float>(f), r = static_cast<float>(f - h) * 3.14159265f;
      float s, c;
      sincospif(h, &s, &c);
      const float c1 = __fmaf_rn(-s, r, c), s1 = __fmaf_rn(c, r, s);
      cs[e] = c1 * p.factor;
      sg[e] = (p.inter || lead ? -s1 : s1) * p.factor;
    }
  }
  // the lane that holds this lane's partners
  const int partner = sub * LPR + (p.inter || !turned ? l : lead ? l + half / 8 : l - half / 8);

  // One loop per kind of row, a row per turn with the next two in flight: short loops, since
  // the three kinds unrolled side by side ran at a quarter of this speed (the code of a turn
  // left the schedulers' instruction caches).
  auto each = [&](const void* src, const int64_t (&st)[3], int h0, int h1, auto&& row_of) {
    const char* base = static_cast<const char*>(src) + 2 * (b * st[0] + i * st[2] + d0);
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
  each(p.q, p.qs, r0, min(r1, p.Hq), [&](int h, const uint4& x) {
    float f[8], o[8], y[8];
    Vec16<DT>::unpack(x, f);
    partners(x, f, o);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __fmaf_rn(f[e], cs[e], o[e] * sg[e]);
    uint4 w = x;
    if (live) w = make_uint4(pack16<DT>(y[0], y[1]), pack16<DT>(y[2], y[3]), pack16<DT>(y[4], y[5]),
                             pack16<DT>(y[6], y[7]));
    if (here)
      *reinterpret_cast<uint4*>(static_cast<char*>(p.q_out) +
                                2 * (b * p.qos[0] + h * p.qos[1] + i * p.qos[2] + d0)) = w;
  });
  each(p.k, p.ks, max(r0 - p.Hq, 0), min(r1 - p.Hq, p.Hkv), [&](int h, const uint4& x) {
    float f[8], o[8], sc[8];
    Vec16<DT>::unpack(x, f);
    partners(x, f, o);
    const int64_t si = b * p.kss[0] + h * p.kss[1] + d0 * p.kss[2];
    if (p.ks_vec && p.s_dt == HQ_DTYPE_F16) {
      Vec16<HQ_DTYPE_F16>::unpack(*reinterpret_cast<const uint4*>(static_cast<const __half*>(p.ksc) + si), sc);
    } else if (p.ks_vec) {
      Vec16<HQ_DTYPE_F32>::unpack(*reinterpret_cast<const uint4*>(static_cast<const float*>(p.ksc) + si), sc);
      Vec16<HQ_DTYPE_F32>::unpack(*reinterpret_cast<const uint4*>(static_cast<const float*>(p.ksc) + si + 4), sc + 4);
    } else {
#pragma unroll 1
      for (int e = 0; e < 8; ++e) {
        const float v = p.s_dt == HQ_DTYPE_F16 ? __half2float(static_cast<const __half*>(p.ksc)[si + e * p.kss[2]])
                                               : static_cast<const float*>(p.ksc)[si + e * p.kss[2]];
#pragma unroll
        for (int g = 0; g < 8; ++g) sc[g] = g == e ? v : sc[g];
      }
    }
    // |error of t| <= (|x| + |o|) / scale 2^-21 + 2^-15 for |t| < 128
    float t[8];
    uint32_t near = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float rs;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rs) : "f"(sc[e]));
      t[e] = __fmaf_rn(f[e], cs[e], o[e] * sg[e]) * rs;
      const float k0 = rintf(t[e]);
      const float slack = __fmaf_rn((fabsf(f[e]) + fabsf(o[e])) * rs, p.slack, 3.0517578e-5f);
      if (!(fabsf(t[e] - k0) + slack < 0.5f) && !(fabsf(t[e]) > 128.0f)) near |= 1u << e;
      t[e] = fminf(fmaxf(k0, -127.0f), 127.0f) + 12582912.0f;  // the code in the low byte
    }
    if (write) {
      uint32_t lo = pack_low_bytes(f2_make(t[0], t[1]), f2_make(t[2], t[3]));
      uint32_t hi = pack_low_bytes(f2_make(t[4], t[5]), f2_make(t[6], t[7]));
      while (near) {
        const int e = __ffs(near) - 1;
        near &= near - 1;
        float fe = 0.0f, oe = 0.0f, se = 1.0f;
#pragma unroll
        for (int g = 0; g < 8; ++g)
          if (g == e) {
            fe = f[g];
            oe = o[g];
            se = sc[g];
          }
        const int j = j0 + (p.inter ? e / 2 : e);
        const uint32_t c = exact_code(fe, oe, p.inter ? !(e & 1) : lead, turned,
                                      turned ? pos * static_cast<double>(p.inv_freq[j]) : 0.0,
                                      p.factor, se) & 0xff;
        const int at = 8 * (e & 3);
        if (e < 4) lo = (lo & ~(0xffu << at)) | c << at;
        else hi = (hi & ~(0xffu << at)) | c << at;
      }
      *reinterpret_cast<uint2*>(p.kc + b * p.cs[0] + h * p.cs[1] + row * p.cs[2] + d0) = make_uint2(lo, hi);
    }
  });
  each(p.v, p.vs, max(r0 - p.Hq - p.Hkv, 0), r1 - p.Hq - p.Hkv, [&](int h, const uint4& x) {
    float f[8];
    Vec16<DT>::unpack(x, f);
    uint32_t a = absmax_x2<DT>(absmax_x2<DT>(x.x, x.y), absmax_x2<DT>(x.z, x.w));
    float m = absmax_of_x2<DT>(a);
#pragma unroll
    for (int o = LPR / 2; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (write) {
      const Quantizer qz = Quantizer::from_amax16(m);
      // the branch-free exact quotient of 16-bit inputs
      const F2 ns = f2_make(-qz.scale, -qz.scale), rc = f2_make(qz.rcp, qz.rcp);
      F2 y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = round_magic(quot_pair(f2_make(f[2 * e], f[2 * e + 1]), ns, rc));
      *reinterpret_cast<uint2*>(p.vc + b * p.cs[0] + h * p.cs[1] + row * p.cs[2] + d0) =
          make_uint2(pack_low_bytes(y[0], y[1]), pack_low_bytes(y[2], y[3]));
      if (l == 0) {
        const int64_t so = b * p.vss[0] + h * p.vss[1] + row * p.vss[2];
        if (p.s_dt == HQ_DTYPE_F16) static_cast<__half*>(p.vsc)[so] = __float2half_rn(qz.scale);
        else static_cast<float*>(p.vsc)[so] = qz.scale;
      }
    }
  });
}

template <int DT, int D>
int launch16(Params p, int B, cudaStream_t st) {
  constexpr int TPW = 32 / (D / 8);
  p.tokens = static_cast<int64_t>(B) * p.S;
  const int rows = p.Hq + 2 * p.Hkv;
  const int64_t warps = (p.tokens + TPW - 1) / TPW;
  // a token's rows stay with one warp (its cos and sin made once) as long as that leaves 16
  // warps per SM; below, they are split, down to one row per warp
  const int64_t want = std::max<int64_t>(1, 16LL * current_sm_count() / warps);
  const int groups = static_cast<int>(std::min<int64_t>(rows, want));
  p.rows_per_block = (rows + groups - 1) / groups;
  p.groups = (rows + p.rows_per_block - 1) / p.rows_per_block;
  const size_t es = p.s_dt == HQ_DTYPE_F16 ? 2 : 4;
  p.ks_vec = p.kss[2] == 1 && reinterpret_cast<uintptr_t>(p.ksc) % 16 == 0 &&
             p.kss[0] * es % 16 == 0 && p.kss[1] * es % 16 == 0;
  p.slack = fmaxf(1.0f, fabsf(p.factor)) * 4.76837158e-7f;  // 2^-21
  const int64_t blocks = (warps * p.groups + kThreads16 / 32 - 1) / (kThreads16 / 32);
  if (blocks > 0x7fffffff) return HQ_ERR_UNSUPPORTED;
  rope_append16_kernel<DT, D><<<static_cast<unsigned>(blocks), kThreads16, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HQ_OK : static_cast<int>(e);
}

// ---------------------------------------------------------------- any type and rotary size
template <int DT, int D>
int launch(Params p, int B, cudaStream_t st) {
  const int64_t tokens = static_cast<int64_t>(B) * p.S;
  const int rows = p.Hq + 2 * p.Hkv;
  // one block per token when that fills the GPU, else the token's rows over several blocks
  const int64_t want = std::max<int64_t>(1, 2LL * current_sm_count() / tokens);
  const int groups = static_cast<int>(std::min<int64_t>((rows + kWarps - 1) / kWarps, want));
  p.rows_per_block = (rows + groups - 1) / groups;
  const dim3 grid(static_cast<unsigned>(tokens), (rows + p.rows_per_block - 1) / p.rows_per_block);
  rope_append_kernel<DT, D><<<grid, kThreads, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HQ_OK : static_cast<int>(e);
}

template <int DT>
int dispatch(const Params& p, int B, cudaStream_t st) {
  if constexpr (DT != HQ_DTYPE_F32) {
    if (p.rot % 16 == 0) {
      if (p.D == 64) return launch16<DT, 64>(p, B, st);
      if (p.D == 128) return launch16<DT, 128>(p, B, st);
      return launch16<DT, 256>(p, B, st);
    }
  }
  if (p.D == 64) return launch<DT, 64>(p, B, st);
  if (p.D == 128) return launch<DT, 128>(p, B, st);
  return launch<DT, 256>(p, B, st);
}

}  // namespace rope
}  // namespace hq

using namespace hq;

extern "C" int hq_rope_append_kv(
    const void* q, const void* k_new, const void* v_new, int x_dtype, const int64_t q_strides[4],
    const int64_t k_strides[4], const int64_t v_strides[4], int B, int Hq, int Hkv, int S_new,
    int D, const float* inv_freq, int rotary_dim, int interleaved, float factor, const int* lens,
    const int* n_new, const int* pos_offset, const void* k_scale, int scale_dtype,
    const int64_t ksc_strides[3], int8_t* k_cache, int8_t* v_cache, const int64_t kv_strides[3],
    void* v_scale, const int64_t vsc_strides[3], int capacity, void* q_out,
    const int64_t qo_strides[4], int* status, hq_stream_t stream) {
  if (!q || !k_new || !v_new || !lens || !k_scale || !k_cache || !v_cache || !v_scale || !q_out ||
      !q_strides || !k_strides || !v_strides || !ksc_strides || !kv_strides || !vsc_strides ||
      !qo_strides || (rotary_dim > 0 && !inv_freq) || B < 0 || Hq < 0 || Hkv <= 0 || S_new < 0 ||
      capacity < 0 || rotary_dim < 0 || rotary_dim > D || rotary_dim % 2)
    return HQ_ERR_INVALID_ARGUMENT;
  if ((D != 64 && D != 128 && D != 256) ||
      (x_dtype != HQ_DTYPE_BF16 && x_dtype != HQ_DTYPE_F16 && x_dtype != HQ_DTYPE_F32) ||
      (scale_dtype != HQ_DTYPE_F32 && scale_dtype != HQ_DTYPE_F16))
    return HQ_ERR_UNSUPPORTED;
  auto al = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
  const int unit = x_dtype == HQ_DTYPE_F32 ? 4 : 8;  // 16-byte rows
  const int64_t* in[4] = {q_strides, k_strides, v_strides, qo_strides};
  for (const int64_t* s : in)
    if (s[3] != 1 || s[0] % unit || s[1] % unit || s[2] % unit) return HQ_ERR_INVALID_ARGUMENT;
  if (!al(q) || !al(k_new) || !al(v_new) || !al(q_out) || !al(k_cache) || !al(v_cache) ||
      kv_strides[0] % 16 || kv_strides[1] % 16 || kv_strides[2] % 16)
    return HQ_ERR_INVALID_ARGUMENT;
  // what is written has rows of its own for every sequence, head and token
  const int64_t* written[3] = {qo_strides, kv_strides, vsc_strides};
  const int extent[3][3] = {{B, Hq, S_new}, {B, Hkv, capacity}, {B, Hkv, capacity}};
  for (int t = 0; t < 3; ++t)
    for (int i = 0; i < 3; ++i)
      if (extent[t][i] > 1 && written[t][i] == 0) return HQ_ERR_INVALID_ARGUMENT;
  if (B == 0 || S_new == 0) return HQ_OK;
  if (static_cast<int64_t>(B) * S_new > 0x7fffffff) return HQ_ERR_UNSUPPORTED;
  rope::Params p{};
  p.q = q;
  p.k = k_new;
  p.v = v_new;
  p.q_out = q_out;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = q_strides[i];
    p.ks[i] = k_strides[i];
    p.vs[i] = v_strides[i];
    p.qos[i] = qo_strides[i];
    p.kss[i] = ksc_strides[i];
    p.cs[i] = kv_strides[i];
    p.vss[i] = vsc_strides[i];
  }
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.S = S_new;
  p.D = D;
  p.inv_freq = inv_freq;
  p.rot = rotary_dim;
  p.inter = interleaved;
  p.factor = factor;
  p.lens = lens;
  p.n_new = n_new;
  p.pos_offset = pos_offset;
  p.ksc = k_scale;
  p.s_dt = scale_dtype;
  p.kc = k_cache;
  p.vc = v_cache;
  p.vsc = v_scale;
  p.cap = capacity;
  p.status = status;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (x_dtype == HQ_DTYPE_BF16) return rope::dispatch<HQ_DTYPE_BF16>(p, B, st);
  if (x_dtype == HQ_DTYPE_F16) return rope::dispatch<HQ_DTYPE_F16>(p, B, st);
  return rope::dispatch<HQ_DTYPE_F32>(p, B, st);
}
