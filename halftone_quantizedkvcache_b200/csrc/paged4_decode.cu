// Decode attention over a paged 4-bit cache (paged4.cuh), one new token per sequence, lengths on the
// device (sm_100a).
//
// All sequences, kv heads and tokens are one line of 32-token tiles; every warp takes an equal run of
// it, with an online softmax of its own and no word to the other warps.  Units (sequence, kv head, up
// to 4 NT query rows) that end inside one warp's run are written by it, the others leave partial
// states (m, l, o) that join_kernel puts together in the order of the line.
//
// Bound by the cache's bytes and, close behind, by issue slots: 144 bytes a token and head are 256
// codes to unpack.  Both products take the codes as the 16-row operand of mma.sync m16n8k16 (bf16),
// query rows in pairs of columns (upper and lower part of a 16-bit split):
//   * Q K^T: a code is 128 + c (its 4 bits under bf16's exponent), no subtraction: the accumulators
//     start at -136 sum(q), formed per unit by the same instruction.  Per group of 32 channels the
//     products are exact and the sum is float32; the group's scale multiplies it in float32.
//   * P V: codes as 128 + c - 136 (exact), p times the token's group scale as a bf16 pair (16 bits,
//     bf16's range: V scales of any size), transposed in registers by movmatrix.
// Copies: every warp has its own ring of stages filled by bulk copies, one per page, side and kind.
//
// No sum is in fewer than 32 bits; q's and p's splits keep 16 bits (2^-17 of each).
#include <algorithm>
#include <atomic>

#include "paged4.cuh"

namespace hq {
int current_sm_count();

namespace p4 {

constexpr int kTile = 32;                 // tokens
constexpr int kMaxSeqs = 1024;
constexpr int kPartRow = kD + 4;          // m, l, two pad words, o
constexpr int kStageB = 2 * kTile * (kRowB + kScaleB);
constexpr int kOffV = kTile * kRowB, kOffKs = 2 * kTile * kRowB, kOffVs = kOffKs + kTile * kScaleB;

struct DecodeParams {
  Pages pg;
  const void* q;
  int64_t qs[2];
  int B, Hkv, nrep, n_rt;                 // row tiles of a kv head's rows
  const int* lens;
  float qk_scale;                         // sm_scale log2(e)
  void* out;
  int64_t os[2];
  float* part;
  int* cum;                               // for join_kernel: first tile of every sequence
  int workers, min_tiles;
  int* status;
};

template <int NT>
struct Cfg {
  // NT 1: 16 warps of 128 registers; NT 2 (twice the accumulators): 8 of 255
  static constexpr int kWarps = NT == 1 ? 16 : 8;
  static constexpr int kStages = NT == 1 ? 3 : 6;
  static constexpr int kRows = 4 * NT;
  static constexpr int kOffBar = kWarps * kStages * kStageB;
  static constexpr int kOffCum = kOffBar + 8 * kWarps * kStages;
  static constexpr int smem(int B) { return kOffCum + 4 * (2 * B + 1); }
  static_assert(smem(kMaxSeqs) <= 232448, "one block per SM");
};

__device__ __forceinline__ int seq_len(const DecodeParams& p, int b) {
  return min(max(p.lens[b], 0), p.pg.max_pages << p.pg.page_log);
}
__device__ __forceinline__ int tiles_of(int len) { return max(1, (len + kTile - 1) / kTile); }

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
// nibbles i and i + 4 of w under the exponent of 128
template <int I>
__device__ __forceinline__ uint32_t biased(uint32_t w) {
  return ((w >> (4 * I)) & 0x000f000fu) | 0x43004300u;
}
__device__ __forceinline__ uint32_t sub136(uint32_t x) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(0x43084308u));
  return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&x);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 half2_of(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// A place on the line of tiles.
struct Cursor {
  int line, end;
  int e, idx, first;                      // sequence, unit within it, the unit's first tile
  int len, nt;
};
__device__ __forceinline__ void enter(Cursor& c, const int* lens, int e) {
  c.e = e;
  c.len = lens[e];
  c.nt = tiles_of(c.len);
}
// to the next tile; units per sequence `per`
__device__ __forceinline__ void step(Cursor& c, const int* lens, int per) {
  if (++c.line == c.first + c.nt && c.line < c.end) {
    c.first = c.line;
    if (++c.idx == per) {
      c.idx = 0;
      enter(c, lens, c.e + 1);
    }
  }
}

template <int NT>
__global__ void __launch_bounds__(32 * Cfg<NT>::kWarps, 1) decode_kernel(const __grid_constant__ DecodeParams p, int q_dt) {
  using C = Cfg<NT>;
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n8 = lane >> 2, c4 = lane & 3;
  unsigned char* ring = smem + warp * C::kStages * kStageB;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar) + warp * C::kStages;
  int* cum = reinterpret_cast<int*>(smem + C::kOffCum);
  int* lens = cum + p.B + 1;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (lane == 0)
    for (int i = 0; i < C::kStages; ++i) mbar_init(&full[i], 1);
  fence_mbar_init();
  const int per = p.Hkv * p.n_rt;
  for (int b = tid; b < p.B; b += 32 * C::kWarps) lens[b] = seq_len(p, b);
  __syncthreads();
  if (warp == 0) {
    int run = 0;
    if (lane == 0) cum[0] = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      int x = b0 + lane < p.B ? tiles_of(lens[b0 + lane]) * per : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (b0 + lane < p.B) cum[b0 + lane + 1] = run + x;
      run += __shfl_sync(0xffffffffu, x, 31);
    }
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int b = tid; b <= p.B; b += 32 * C::kWarps) p.cum[b] = cum[b];
  const int total = cum[p.B];
  const int chunk = max(p.min_tiles, (total + p.workers - 1) / p.workers);
  // neighbouring runs on different SMs
  const int worker = warp * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x);
  Cursor cur{};
  cur.line = static_cast<int>(min(static_cast<int64_t>(worker) * chunk, static_cast<int64_t>(total)));
  cur.end = static_cast<int>(min(static_cast<int64_t>(cur.line) + chunk, static_cast<int64_t>(total)));
  if (cur.line >= cur.end) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  {
    int lo = 0, hi = p.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cum[mid] <= cur.line) lo = mid; else hi = mid - 1;
    }
    enter(cur, lens, lo);
    cur.idx = static_cast<uint32_t>(cur.line - cum[lo]) / static_cast<uint32_t>(cur.nt);
    cur.first = cum[lo] + cur.idx * cur.nt;
  }

  // ---- the copies' cursor, up to kStages tiles ahead
  Cursor ahead = cur;
  int win_e = -1, win = 0, ids = 0;       // 32 page numbers of sequence win_e from entry `win` on
  int issued = 0;
  auto issue = [&]() {
    if (ahead.line >= ahead.end) return;
    const int st = issued % C::kStages;
    const int tok = (ahead.line - ahead.first) * kTile;
    const int pi = tok >> p.pg.page_log;
    if (win_e != ahead.e || pi < win || pi >= win + 32) {
      win_e = ahead.e;
      win = pi & ~31;
      const int at = win + lane;
      ids = at << p.pg.page_log < ahead.len ? p.pg.tables[win_e * p.pg.tstride + at] : -1;
    }
    const int kvh = p.n_rt == 1 ? ahead.idx : ahead.idx / p.n_rt;
    const int here = min(p.pg.page, kTile);  // tokens of a page in the tile
    unsigned char* s = ring + st * kStageB;
    uint32_t bytes = 0;
    int page[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      page[i] = -1;
      if (i * here < kTile && tok + i * here < ahead.len) {
        page[i] = __shfl_sync(0xffffffffu, ids, (pi - win + i) & 31);
        if (page[i] >= 0 && page[i] < p.pg.n_pages) {
          bytes += 2 * here * (kRowB + kScaleB);
        } else {
          page[i] = -1;
          if (lane == 0) report_error(p.status, HQ_ERR_INVALID_ARGUMENT);
        }
      }
    }
    if (lane == 0) {
      if (bytes) mbar_arrive_expect_tx(&full[st], bytes);
      else mbar_arrive(&full[st]);
      const int off = tok & (p.pg.page - 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (page[i] < 0) continue;
        const int64_t co = page[i] * p.pg.cp + kvh * p.pg.ch + off * kRowB;
        const int64_t so = page[i] * p.pg.sp + kvh * p.pg.sh + off * 4;
        bulk_g2s(s + i * here * kRowB, p.pg.k + co, here * kRowB, &full[st]);
        bulk_g2s(s + kOffKs + i * here * kScaleB, p.pg.ksc + so, here * kScaleB, &full[st]);
        bulk_g2s(s + kOffV + i * here * kRowB, p.pg.v + co, here * kRowB, &full[st]);
        bulk_g2s(s + kOffVs + i * here * kScaleB, p.pg.vsc + so, here * kScaleB, &full[st]);
      }
    }
    ++issued;
    step(ahead, lens, per);
  };
  __syncwarp();
#pragma unroll 1
  for (int i = 0; i < C::kStages; ++i) issue();

  // tokens of this lane's slots n8 and n8 + 8 of a block of 16 (Q K^T's rows, P's entries)
  const int e1 = n8 & 1, slot_tok = 4 * e1 + ((n8 >> 1) ^ e1);
  // V: rows n8 (and n8 + 8) are channels of chunk vj, half vh
  const int vj = n8 & 3, vh = n8 >> 2;
  const uint32_t vsel = vh ? 0x7632u : 0x5410u;
  // K rows of slots: byte offset of chunk c4 of token slot_tok; V: chunk vj of tokens c4, 4 + (c4 ^ 1)
  const int k_off = slot_tok * kRowB + 16 * (c4 ^ (slot_tok & 2));
  const int va = c4, vb = 4 + (c4 ^ 1);
  const int va_off = kOffV + va * kRowB + 16 * (vj ^ (va & 2)), vb_off = kOffV + vb * kRowB + 16 * (vj ^ (vb & 2));

  int done = 0;
  bool ok = true;
#pragma unroll 1
  while (ok && cur.line < cur.end) {
    // ---- a piece: tiles t0 .. t1 - 1 of one unit
    const int t0 = cur.line - cur.first, t1 = min(cur.nt, t0 + cur.end - cur.line);
    const int kvh = p.n_rt == 1 ? cur.idx : cur.idx / p.n_rt;
    const int row0 = (cur.idx - kvh * p.n_rt) * C::kRows;
    const int b = cur.e, len = cur.len;
    const int slot = t0 == 0 && t1 == cur.nt ? -1 : cur.e * per + cur.idx + worker;
    // B fragments of q: column n8 is the upper (n8 even) or lower part of row 4 nt + n8 / 2
    uint32_t bq[NT][4][2][2];
    float corr[NT][4][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row0 + 4 * nt + (n8 >> 1);
      const bool real = r < p.nrep;
      const char* row = static_cast<const char*>(p.q) + 2 * (b * p.qs[0] + (kvh * p.nrep + r) * p.qs[1] + 8 * c4);
      uint4 raw[4];
#pragma unroll
      for (int g = 0; g < 4; ++g)
        raw[g] = real ? *reinterpret_cast<const uint4*>(row + 64 * g) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float f[8];
        if (q_dt == HQ_DTYPE_BF16) Vec16<HQ_DTYPE_BF16>::unpack(raw[g], f);
        else Vec16<HQ_DTYPE_F16>::unpack(raw[g], f);
        if (n8 & 1) {
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] -= __bfloat162float(__float2bfloat16_rn(f[e]));
        }
        // channels 8 c4 + 2 m, + 4 and 8 c4 + 2 m + 1, + 5
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          bq[nt][g][m][0] = pack_bf16(f[2 * m], f[2 * m + 4]);
          bq[nt][g][m][1] = pack_bf16(f[2 * m + 1], f[2 * m + 5]);
        }
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        constexpr uint32_t kM136 = 0xc308c308u;
#pragma unroll
        for (int m = 0; m < 2; ++m) mma_bf16(s, kM136, kM136, kM136, kM136, bq[nt][g][m][0], bq[nt][g][m][1]);
        corr[nt][g][0] = s[0];
        corr[nt][g][1] = s[1];
      }
    }
    float m_run[NT], l_run[NT], o[NT][4][2][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m_run[nt] = -INFINITY;
      l_run[nt] = 0.0f;
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][g][m][e] = 0.0f;
    }

#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      const int st = done % C::kStages;
      ok = mbar_wait(&full[st], (done / C::kStages) & 1);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      ++done;
      const unsigned char* s = ring + st * kStageB;
      const int left = len - t * kTile;   // tokens of the tile that exist
      float sc[NT][2][2];
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const unsigned char* kr = s + blk * 16 * kRowB + k_off;
        const uint4 w0 = *reinterpret_cast<const uint4*>(kr);
        const uint4 w1 = *reinterpret_cast<const uint4*>(kr + 8 * kRowB);
        const uint32_t a0[4] = {w0.x, w0.y, w0.z, w0.w}, a1[4] = {w1.x, w1.y, w1.z, w1.w};
        const unsigned char* ks = s + kOffKs + (blk * 16 + slot_tok) * kScaleB;
        const uint2 u0 = *reinterpret_cast<const uint2*>(ks);
        const uint2 u1 = *reinterpret_cast<const uint2*>(ks + 8 * kScaleB);
        const float2 k00 = half2_of(u0.x), k01 = half2_of(u0.y), k10 = half2_of(u1.x), k11 = half2_of(u1.y);
        const float s0[4] = {k00.x, k00.y, k01.x, k01.y}, s1[4] = {k10.x, k10.y, k11.x, k11.y};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[nt][blk][0] = sc[nt][blk][1] = 0.0f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const uint32_t x0 = biased<0>(a0[g]), x1 = biased<1>(a0[g]), x2 = biased<2>(a0[g]), x3 = biased<3>(a0[g]);
          const uint32_t y0 = biased<0>(a1[g]), y1 = biased<1>(a1[g]), y2 = biased<2>(a1[g]), y3 = biased<3>(a1[g]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float c[4] = {corr[nt][g][0], corr[nt][g][1], corr[nt][g][0], corr[nt][g][1]};
            mma_bf16(c, x0, y0, x1, y1, bq[nt][g][0][0], bq[nt][g][0][1]);
            mma_bf16(c, x2, y2, x3, y3, bq[nt][g][1][0], bq[nt][g][1][1]);
            sc[nt][blk][0] = __fmaf_rn(s0[g], c[0] + c[1], sc[nt][blk][0]);
            sc[nt][blk][1] = __fmaf_rn(s1[g], c[2] + c[3], sc[nt][blk][1]);
          }
        }
        const int tk = blk * 16 + slot_tok;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          sc[nt][blk][0] = tk < left ? sc[nt][blk][0] * p.qk_scale : -INFINITY;
          sc[nt][blk][1] = tk + 8 < left ? sc[nt][blk][1] * p.qk_scale : -INFINITY;
        }
      }
      // ---- online softmax
      float pr[NT][2][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float mt = fmaxf(fmaxf(sc[nt][0][0], sc[nt][0][1]), fmaxf(sc[nt][1][0], sc[nt][1][1]));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 4));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 8));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 16));
        if (__any_sync(0xffffffffu, mt > m_run[nt])) {
          const float m_new = fmaxf(m_run[nt], mt);
          const float alpha = m_run[nt] == m_new ? 1.0f : ex2(m_run[nt] - m_new);
          m_run[nt] = m_new;
          l_run[nt] *= alpha;
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nt][g][m][e] *= alpha;
        }
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float x = sc[nt][blk][i];
            pr[nt][blk][i] = x == -INFINITY ? 0.0f : ex2(x - m_run[nt]);
            l_run[nt] += pr[nt][blk][i];
          }
      }
      // ---- P V
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const unsigned char* v0 = s + blk * 16 * kRowB;
        const uint4 ta = *reinterpret_cast<const uint4*>(v0 + va_off), tb = *reinterpret_cast<const uint4*>(v0 + vb_off);
        const uint4 tc = *reinterpret_cast<const uint4*>(v0 + va_off + 8 * kRowB);
        const uint4 td = *reinterpret_cast<const uint4*>(v0 + vb_off + 8 * kRowB);
        const uint32_t wa[4] = {ta.x, ta.y, ta.z, ta.w}, wb[4] = {tb.x, tb.y, tb.z, tb.w};
        const uint32_t wc[4] = {tc.x, tc.y, tc.z, tc.w}, wd[4] = {td.x, td.y, td.z, td.w};
        const int tk = blk * 16 + slot_tok;
        const unsigned char* vs = s + kOffVs + tk * kScaleB;
        uint2 u0 = *reinterpret_cast<const uint2*>(vs), u1 = *reinterpret_cast<const uint2*>(vs + 8 * kScaleB);
        if (tk >= left) u0 = make_uint2(0, 0);      // what no token wrote may be anything
        if (tk + 8 >= left) u1 = make_uint2(0, 0);
        const float2 k00 = half2_of(u0.x), k01 = half2_of(u0.y), k10 = half2_of(u1.x), k11 = half2_of(u1.y);
        const float s0[4] = {k00.x, k00.y, k01.x, k01.y}, s1[4] = {k10.x, k10.y, k11.x, k11.y};
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const uint32_t x = prmt(wa[g], wb[g], vsel), y = prmt(wc[g], wd[g], vsel);
          const uint32_t x0 = sub136(biased<0>(x)), x1 = sub136(biased<1>(x)), x2 = sub136(biased<2>(x)), x3 = sub136(biased<3>(x));
          const uint32_t y0 = sub136(biased<0>(y)), y1 = sub136(biased<1>(y)), y2 = sub136(biased<2>(y)), y3 = sub136(biased<3>(y));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float p0 = pr[nt][blk][0] * s0[g], p1 = pr[nt][blk][1] * s1[g];
            const uint32_t hi = pack_bf16(p0, p1);
            const uint32_t lo = pack_bf16(p0 - __uint_as_float(hi << 16), p1 - __uint_as_float(hi & 0xffff0000u));
            const uint32_t b0 = transpose8(prmt(hi, lo, 0x5410u)), b1 = transpose8(prmt(hi, lo, 0x7632u));
            mma_bf16(o[nt][g][0], x0, x1, y0, y1, b0, b1);
            mma_bf16(o[nt][g][1], x2, x3, y2, y3, b0, b1);
          }
        }
      }
      __syncwarp();
      issue();
      step(cur, lens, per);
    }
    if (!ok) break;

    // ---- the piece's rows: lane (n8, c4) holds row 4 nt + c4, channels 32 g + 8 vj + 4 vh + 2 m, + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float l = l_run[nt];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const int r = row0 + 4 * nt + c4;
      if (r >= p.nrep) continue;
      const int ch = 8 * vj + 4 * vh;
      if (slot < 0) {
        const float inv = l <= 0.0f ? 0.0f : 1.0f / l;  // (a NaN stays)
        char* dst = static_cast<char*>(p.out) + 2 * (b * p.os[0] + (kvh * p.nrep + r) * p.os[1] + ch);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          uint32_t w[2];
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const float x = (o[nt][g][m][0] + o[nt][g][m][1]) * inv, y = (o[nt][g][m][2] + o[nt][g][m][3]) * inv;
            if (q_dt == HQ_DTYPE_BF16) {
              w[m] = pack_bf16(x, y);
            } else {
              const __half2 h = __floats2half2_rn(x, y);
              w[m] = *reinterpret_cast<const uint32_t*>(&h);
            }
          }
          *reinterpret_cast<uint2*>(dst + 64 * g) = make_uint2(w[0], w[1]);
        }
      } else {
        float* dst = p.part + (static_cast<int64_t>(slot) * C::kRows + 4 * nt + c4) * kPartRow;
        if (n8 == 0) *reinterpret_cast<float2*>(dst) = make_float2(m_run[nt], l);
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4*>(dst + 4 + 32 * g + ch) =
              make_float4(o[nt][g][0][0] + o[nt][g][0][1], o[nt][g][0][2] + o[nt][g][0][3],
                          o[nt][g][1][0] + o[nt][g][1][1], o[nt][g][1][2] + o[nt][g][1][3]);
      }
    }
  }
  if (!ok) {
    report_error(p.status, HQ_ERR_DEVICE_TIMEOUT);
    for (int i = done; i < issued; ++i) mbar_wait(&full[i % C::kStages], (i / C::kStages) & 1);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// One block per output row (sequence, q head): warp w joins pieces w, w + 4, .. of the row's unit, a
// lane 4 channels, then warp 0 the warps' sums; always in the same order.
constexpr int kJoinWarps = 4;
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const __grid_constant__ DecodeParams p, int q_dt, int rows) {
  __shared__ float4 sum[kJoinWarps][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.x % (p.Hkv * p.nrep), b = blockIdx.x / (p.Hkv * p.nrep);
  const int kvh = h / p.nrep, hr = h - kvh * p.nrep, rt = hr / rows;
  const int per = p.Hkv * p.n_rt, idx = kvh * p.n_rt + rt;
  const int total = p.cum[p.B], chunk = max(p.min_tiles, (total + p.workers - 1) / p.workers);
  const int nt = (p.cum[b + 1] - p.cum[b]) / per;
  const int first = p.cum[b] + idx * nt, w0 = first / chunk, w1 = (first + nt - 1) / chunk;
  if (w0 == w1) return;                   // written by its only worker
  const float* at = p.part + (static_cast<int64_t>(b * per + idx + w0) * rows + hr - rt * rows) * kPartRow;
  const int64_t dist = static_cast<int64_t>(rows) * kPartRow;
  float M = -INFINITY, L = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](float m, float l, const float4& x) {
    const float top = fmaxf(M, m);
    const float f0 = M == -INFINITY ? 0.0f : exp2f(M - top), f1 = m == -INFINITY ? 0.0f : exp2f(m - top);
    M = top;
    L = L * f0 + l * f1;
    acc.x = acc.x * f0 + x.x * f1;
    acc.y = acc.y * f0 + x.y * f1;
    acc.z = acc.z * f0 + x.z * f1;
    acc.w = acc.w * f0 + x.w * f1;
  };
#pragma unroll 4
  for (int i = warp; i <= w1 - w0; i += kJoinWarps) {
    const float* x = at + i * dist;
    const float2 ml = *reinterpret_cast<const float2*>(x);
    add(ml.x, ml.y, *reinterpret_cast<const float4*>(x + 4 + 4 * lane));
  }
  sum[warp][lane] = acc;
  if (lane == 0) sum[warp][32] = make_float4(M, L, 0.0f, 0.0f);
  __syncthreads();
  if (warp) return;
#pragma unroll
  for (int i = 1; i < kJoinWarps; ++i) {
    const float4 ml = sum[i][32];
    add(ml.x, ml.y, sum[i][lane]);
  }
  const float inv = L <= 0.0f ? 0.0f : 1.0f / L;
  char* dst = static_cast<char*>(p.out) + 2 * (b * p.os[0] + h * p.os[1] + 4 * lane);
  uint2 w;
  if (q_dt == HQ_DTYPE_BF16) {
    w = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
  } else {
    const __half2 x = __floats2half2_rn(acc.x * inv, acc.y * inv), y = __floats2half2_rn(acc.z * inv, acc.w * inv);
    w = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
  *reinterpret_cast<uint2*>(dst) = w;
}

// ---------------------------------------------------------------- host
struct DecodePlan {
  int nt, n_rt, grid, workers;
  size_t cum_bytes, bytes;
};
inline size_t align256(size_t n) { return (n + 255) & ~size_t(255); }
inline bool plan_decode(DecodePlan& pl, int B, int Hkv, int nrep, int64_t cap) {
  if (B > kMaxSeqs || nrep > 128) return false;
  // up to 4 rows a kv head: one column pair each; above, 8 at a time
  pl.nt = nrep <= 4 ? 1 : 2;
  const int rows = 4 * pl.nt;
  pl.n_rt = (nrep + rows - 1) / rows;
  const int64_t units = int64_t(B) * Hkv * pl.n_rt, tiles = units * std::max<int64_t>(1, (cap + kTile - 1) / kTile);
  if (tiles > (int64_t(1) << 30)) return false;
  const int warps = pl.nt == 1 ? Cfg<1>::kWarps : Cfg<2>::kWarps;
  // a block per SM; with few tiles one tile a warp, spread over the SMs
  pl.grid = static_cast<int>(std::min<int64_t>(current_sm_count(), std::max<int64_t>(tiles, 1)));
  pl.workers = pl.grid * warps;
  pl.cum_bytes = align256(sizeof(int) * (B + 1));
  pl.bytes = pl.cum_bytes + align256(sizeof(float) * static_cast<size_t>(units + pl.workers) * rows * kPartRow);
  return true;
}

template <int NT>
int launch_decode(const DecodeParams& p, int q_dt, const DecodePlan& pl, cudaStream_t st) {
  using C = Cfg<NT>;
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = dev >= 0 && dev < 64 ? uint64_t(1) << dev : 0;
  if (!bit || !(ready.load(std::memory_order_acquire) & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(decode_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem(kMaxSeqs));
    if (e != cudaSuccess) return static_cast<int>(e);
    ready.fetch_or(bit, std::memory_order_acq_rel);
  }
  decode_kernel<NT><<<pl.grid, 32 * C::kWarps, C::smem(p.B), st>>>(p, q_dt);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return static_cast<int>(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.B) * p.Hkv * p.nrep);
  cfg.blockDim = dim3(32 * kJoinWarps);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, join_kernel, p, q_dt, C::kRows);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return static_cast<int>(e);
  }
  return HQ_OK;
}

}  // namespace p4
}  // namespace hq

using namespace hq;

extern "C" size_t hq_paged4_decode_workspace_bytes(int B, int Hq, int Hkv, int page_size, int max_pages, int D) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D != p4::kD || page_size < 16 || max_pages < 0) return 0;
  p4::DecodePlan pl{};
  return p4::plan_decode(pl, B, Hkv, Hq / Hkv, int64_t(page_size) * max_pages) ? pl.bytes : 0;
}

extern "C" int hq_paged4_decode(const void* q, int q_dtype, const int64_t q_strides[2], const uint8_t* k_codes,
                                const uint8_t* v_codes, const int64_t code_strides[2], const void* k_scale,
                                const void* v_scale, const int64_t scale_strides[2], int n_pages, int page_size,
                                const int* tables, int64_t table_stride, int max_pages, const int* lens, int B,
                                int Hq, int Hkv, int D, float sm_scale, void* out, const int64_t out_strides[2],
                                void* workspace, size_t workspace_bytes, int* status, hq_stream_t stream) {
  if (B < 0 || Hq <= 0 || Hkv <= 0 || !q_strides || !out_strides) return HQ_ERR_INVALID_ARGUMENT;
  if (D != p4::kD || Hq % Hkv || (q_dtype != HQ_DTYPE_BF16 && q_dtype != HQ_DTYPE_F16)) return HQ_ERR_UNSUPPORTED;
  const int rc = p4::check_pages(k_codes, v_codes, k_scale, v_scale, code_strides, scale_strides, n_pages,
                                 page_size, tables, table_stride, max_pages, B, Hkv);
  if (rc != HQ_OK) return rc;
  if (B == 0) return HQ_OK;
  auto al = [](const void* x, uintptr_t a) { return reinterpret_cast<uintptr_t>(x) % a == 0; };
  if (!q || !out || !lens || !al(q, 16) || !al(out, 8) || q_strides[0] % 8 || q_strides[1] % 8 ||
      out_strides[0] % 4 || out_strides[1] % 4 || (B > 1 && out_strides[0] == 0) || (Hq > 1 && out_strides[1] == 0))
    return HQ_ERR_INVALID_ARGUMENT;
  p4::DecodePlan pl{};
  if (!p4::plan_decode(pl, B, Hkv, Hq / Hkv, int64_t(page_size) * max_pages) || int64_t(B) * Hq > 0x7fffffff)
    return HQ_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < pl.bytes || !al(workspace, 256)) return HQ_ERR_WORKSPACE;
  p4::DecodeParams p{};
  p.pg = p4::make_pages(k_codes, v_codes, k_scale, v_scale, code_strides, scale_strides, n_pages, page_size,
                        tables, table_stride, max_pages);
  p.q = q;
  p.out = out;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = q_strides[i];
    p.os[i] = out_strides[i];
  }
  p.B = B;
  p.Hkv = Hkv;
  p.nrep = Hq / Hkv;
  p.n_rt = pl.n_rt;
  p.lens = lens;
  p.qk_scale = sm_scale * 1.4426950408889634f;
  p.cum = static_cast<int*>(workspace);
  p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.cum_bytes);
  p.workers = pl.workers;
  p.min_tiles = 1;
  p.status = status;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return pl.nt == 1 ? p4::launch_decode<1>(p, q_dtype, pl, st) : p4::launch_decode<2>(p, q_dtype, pl, st);
}
