// Decode attention over int8 caches whose sequences have lengths of their own, for up to 4 query
// rows per kv head (sm_100a): the keys a query sees (all of them, or the window and the sinks)
// as one line of 128-key tiles over all sequences and kv heads, an equal run of it per block.
//
// Bound by the cache's bytes: 256 bytes of codes per key against 4 rows x 256 multiply-adds.
// Both products run on the int8 tensor cores (mma.sync m16n8k32) straight from the codes, so
// nothing is converted: with q' = q k_scale sm_scale log2(e) in 24-bit fixed point per row
// (three balanced base-256 digits, one column each) the scores are exact integers times one
// scale, and P v_scale likewise goes in as three digits; O is float32.  The digits' scale is twice
// the largest p v_scale since a warp's maximum last moved.
//
// A block is 4 warps, 32 keys of a tile each with their own online softmax; two blocks per SM.
// Tiles arrive by TMA into a ring of 3 stages, 128-byte swizzled; two are in flight while one
// is worked on, across the borders of sequences.  A tile inside one run of keys is one box per
// side; the tile in which the sinks end and the window begins is put together from boxes of 8
// keys.  (cp.async of 16 bytes a thread did both with one rule, but under load its issue held
// the warps up for 2400 cycles a tile: 138 us against 108 then at 64 sequences x 4096 keys.)
//
// Measured at 64 sequences x 4096 keys (bf16, 16 q heads over 8 kv heads): 96 us = 5.6 TB/s, 0.86
// of the measured rate.  Short runs pay for their starts: 64 sequences of 64 to 1024 tokens, 34 us =
// 2.1 TB/s, of which a block's start, the joins of its three pieces and their joining kernel take
// two thirds.
#include "decode_common.cuh"
#include "ragged_common.cuh"

namespace hq {
namespace rag {
using namespace dec::mmak;

constexpr int kThreads = 128;
constexpr int kWarps = 4;

template <int NR>
struct RCfg {
  static constexpr int NT = (NR + 1) / 2;                  // n8 tiles, 2 rows each
  // the digit table of q', dead once the fragments are in registers; the warps' sums later
  static constexpr int kOffQtab = kStagesM * 2 * kTileB;   // NT x 1 KB
  static constexpr int kOffWo = kOffQtab;                  // [kWarps][NR][kD]
  static constexpr int kOffLimb = kOffWo + kWarps * NR * kD * 4;  // p' digits, per warp
  static_assert(kOffQtab + NT * 1024 <= kOffLimb, "the table lies inside the sums");
  static constexpr int kOffWm = kOffLimb + kWarps * NT * 256;     // [kWarps][NR] (m, l)
  static constexpr int kOffBar = kOffWm + kWarps * NR * 8;        // [kStagesM] tile arrived
  static constexpr int kOffCum = kOffBar + 32;
  static constexpr int smem(int entries) { return 1024 + kOffCum + 4 * (entries + 1); }
  static_assert(2 * (smem(kMaxEntries) + 1024) <= 233472, "two blocks per SM");
};

struct Maps {
  CUtensorMap k, v;      // boxes of 128 keys
  CUtensorMap k8, v8;    // boxes of 8 keys
  int bm, hm;            // batch and head coordinates' factors (0: one copy for all)
  int inner;             // dimensions (channel, head, key, batch): heads closer than keys
};

template <int NR>
__global__ void __launch_bounds__(kThreads, 2)
    rows_kernel(const __grid_constant__ Params p, const __grid_constant__ Maps maps) {
  using C = RCfg<NR>;
  constexpr int NT = C::NT;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* ring = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* plimb = ring + C::kOffLimb;
  uint32_t* qtab = reinterpret_cast<uint32_t*>(ring + C::kOffQtab);
  float* wo = reinterpret_cast<float*>(ring + C::kOffWo);
  float2* wm = reinterpret_cast<float2*>(ring + C::kOffWm);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + C::kOffBar);
  int* cum = reinterpret_cast<int*>(ring + C::kOffCum);
  __shared__ float red[kWarps][NR];
  __shared__ float qmax_s[NR];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  // dependents may be scheduled; they wait for this grid
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    for (int i = 0; i < kStagesM; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  // zero the p' staging (columns 3 and 7 stay zero)
  for (int i = tid; i < kWarps * NT * 64; i += kThreads) reinterpret_cast<uint32_t*>(plimb)[i] = 0;
  build_cum<128, 8>(p, cum, kThreads);
  Walk walk = walk_start<128, true, 8>(p, cum);
  const Seg& s = p.seg;
  const uint64_t pol = l2_evict_first();

  // ---- the loads' cursor, two tiles ahead
  Piece w{};
  const bool any = walk_next<128, true, 8>(walk, p, cum, w);
  Walk lw = walk;
  Piece lp = w;
  int lt = w.t0 - 1, issued = 0;
  bool more = any;
  int64_t vs0 = lp.b * s.vscb + lp.kvh * s.vsch;
  uint32_t vs_n[3][2] = {};  // V scales of this lane's own keys: this tile, the next two
  // the next tile into stage `st` (nothing past the last), its V scales into the queue's end
  auto issue = [&](int st) {
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      vs_n[0][rb] = vs_n[1][rb];
      vs_n[1][rb] = vs_n[2][rb];
      vs_n[2][rb] = 0u;
    }
    if (more && ++lt >= lp.t1) {
      more = walk_next<128, true, 8>(lw, p, cum, lp);
      lt = lp.t0;
      vs0 = lp.b * s.vscb + lp.kvh * s.vsch;
    }
    if (!more) return;
    ++issued;
    const int v0 = lt * kBN;
    if (tid == 0) {
      unsigned char* kd = ring + st * 2 * kTileB;
      const int head = lp.kvh * maps.hm, z = lp.b * maps.bm;
      const bool one = lp.key.sh == 0 || v0 >= lp.key.nsp || v0 + kBN <= lp.key.nsp;
      const CUtensorMap* mk = one ? &maps.k : &maps.k8;
      const CUtensorMap* mv = one ? &maps.v : &maps.v8;
      if (v0 >= lp.key.nv) {  // an empty sequence: nothing to read, and nothing of it is seen
        mbar_arrive(&full[st]);
      } else {
        mbar_arrive_expect_tx(&full[st], 2 * kTileB);  // (boxes past the cache's end: zeros)
#pragma unroll 1
        for (int i = 0; i < (one ? 1 : kBN); i += 8) {
          const int key = lp.key.key(v0 + i);
          const int x1 = maps.inner ? head : key, x2 = maps.inner ? key : head;
          tma_load_4d(kd + i * kD, mk, 0, x1, x2, z, &full[st], pol);
          tma_load_4d(kd + kTileB + i * kD, mv, 0, x1, x2, z, &full[st], pol);
        }
      }
    }
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      const int v = v0 + warp * 32 + rb * 16 + g + 8 * (t4 & 1);
      if (v < lp.key.nv && !lp.key.padding(v))
        vs_n[2][rb] = load_bits(s.vsc, vs0 + static_cast<int64_t>(lp.key.key(v)) * s.vscs, p.s_dt);
    }
  };

  unsigned char* my_limb = plimb + warp * NT * 256;
  int done = 0;  // tiles worked on
  bool ok = true;
  // a piece's q and K scale of this thread's channel, loaded a piece ahead (bits: a conversion
  // would wait for them)
  const int d = tid;
  uint32_t ksb = 0;
  unsigned short qb[NR] = {};
  auto load_q = [&](const Piece& of) {
    ksb = load_bits(s.ksc, of.b * s.kscb + of.kvh * s.ksch + d * s.kscd, p.s_dt);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      qb[r] = 0;
      if (r < of.rows) {
        const int u = r / p.nrep, h = of.kvh * p.nrep + r - u * p.nrep;
        qb[r] = static_cast<const unsigned short*>(p.q)[of.b * s.qsb + u * s.qsu + h * p.qsh + d];
      }
    }
  };
  if (any) load_q(w);
#pragma unroll 1
  for (int i = 0; i < 2; ++i) issue(i);
  Piece next{};
  bool go = any;
  for (; ok && go; w = next) {
    // ---- q' and its digits; thread owns channel d
    const int rows = w.rows;
    {
      const float ks = scale_of(ksb, p.s_dt);
      float qv[NR];
#pragma unroll
      for (int r = 0; r < NR; ++r)
        qv[r] = p.q_dt == HQ_DTYPE_BF16 ? __uint_as_float(static_cast<uint32_t>(qb[r]) << 16)
                                        : __half2float(__ushort_as_half(qb[r]));
      go = walk_next<128, true, 8>(walk, p, cum, next);
      if (go) load_q(next);
      if (p.q_quant) {  // per-token int8 fake quantization, rounded back to the model dtype
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float m = dec::warp_max(fabsf(qv[r]), 1);
          if (lane == 0) red[warp][r] = m;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const Quantizer qz = Quantizer::from_amax(
              fmaxf(fmaxf(red[0][r], red[1][r]), fmaxf(red[2][r], red[3][r])));
          const float y = static_cast<float>(qz.code(qv[r])) * qz.scale;
          qv[r] = p.q_dt == HQ_DTYPE_BF16 ? __bfloat162float(__float2bfloat16_rn(y))
                                          : __half2float(__float2half_rn(y));
        }
        __syncthreads();
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        qv[r] *= ks * p.qk_scale;
        // (a NaN must not get lost in the maximum)
        const float m = dec::warp_max(qv[r] == qv[r] ? fabsf(qv[r]) : INFINITY, 1);
        if (lane == 0) red[warp][r] = m;
      }
      __syncthreads();
      // B fragments: word (nt, j, hh, lane g * 4 + t4) packs digit g % 4 of row 2 nt + g / 4 at
      // the channels 32 j + 16 hh + 4 t4 + e (what digit 3 and rows past NR hold is multiplied
      // by zero)
      unsigned char* at = reinterpret_cast<unsigned char*>(qtab) +
                          4 * ((d >> 5) * 64 + ((d >> 4) & 1) * 32 + ((d >> 2) & 3)) + (d & 3);
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float qm = fmaxf(fmaxf(red[0][r], red[1][r]), fmaxf(red[2][r], red[3][r]));
        if (tid == 0) qmax_s[r] = qm;
        const float inv = qm > 0.0f ? kLimbMax / qm : 0.0f;
        const int x = max(-static_cast<int>(kLimbMax),
                          min(static_cast<int>(kLimbMax), __float2int_rn(qv[r] * inv)));
        int la, lb, lc;
        limbs24(x, la, lb, lc);
        unsigned char* row = at + 4 * ((r >> 1) * 256 + 4 * (4 * (r & 1)));
        row[0] = static_cast<unsigned char>(la);
        row[16] = static_cast<unsigned char>(lb);
        row[32] = static_cast<unsigned char>(lc);
      }
      __syncthreads();
    }
    uint32_t bq[NT][4][2];
    float f0[NT], f1[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) bq[nt][j][hh] = qtab[(nt << 8) | (j << 6) | (hh << 5) | lane];
      const int r = 2 * nt + (t4 >> 1);
      // (a row whose q' is not finite gives NaN, as its softmax does)
      const float qm = r < NR ? qmax_s[r] : 0.0f;
      const float qsc = qm > 0.0f ? qm / kLimbMax : qm == 0.0f ? 0.0f : qm;
      f0[nt] = (t4 & 1) ? qsc : qsc * 65536.0f;
      f1[nt] = (t4 & 1) ? 0.0f : qsc * 256.0f;
    }
    // running state per n-tile (this lane's row 2 nt + t4 / 2)
    float m_run[NT], l_run[NT], pmax[NT], o_acc[NT][4][2][2];
    int acc[NT][4][2][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m_run[nt] = -INFINITY;
      l_run[nt] = 0.0f;
      pmax[nt] = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int pi = 0; pi < 2; ++pi) {
          o_acc[nt][j][pi][0] = o_acc[nt][j][pi][1] = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[nt][j][pi][e] = 0;
        }
    }
    // the int32 sums of n-tile nt into float (lanes where take)
    auto flush = [&](int nt, bool take) {
      const float ps = pmax[nt] / kLimbMax;
      const float F0 = (t4 & 1) ? ps : ps * 65536.0f;
      const float F1 = (t4 & 1) ? 0.0f : ps * 256.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int pi = 0; pi < 2; ++pi) {
          float lo = F0 * static_cast<float>(acc[nt][j][pi][0]) + F1 * static_cast<float>(acc[nt][j][pi][1]);
          float hi = F0 * static_cast<float>(acc[nt][j][pi][2]) + F1 * static_cast<float>(acc[nt][j][pi][3]);
          lo += __shfl_xor_sync(0xffffffffu, lo, 1);
          hi += __shfl_xor_sync(0xffffffffu, hi, 1);
          if (take) {
            o_acc[nt][j][pi][0] += lo;
            o_acc[nt][j][pi][1] += hi;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][j][pi][e] = 0;
          }
        }
    };

    // the digits' sums stay in int32 for at most this many tiles: 32 keys x 127 x 128 a tile
    int since = 0;
#pragma unroll 1
    for (int t = w.t0; t < w.t1; ++t) {
      const int st = done % kStagesM;
      ok = mbar_wait(&full[st], (done / kStagesM) & 1);
      // (all threads: the stage of the tile before is free for the tile two on)
      if (__syncthreads_or(!ok)) {
        ok = false;
        break;
      }
      ++done;
      issue((st + 2) % kStagesM);
      const float vsf[2] = {scale_of(vs_n[0][0], p.s_dt), scale_of(vs_n[0][1], p.s_dt)};
      const int base = t * kBN + warp * 32, lim = w.key.nv;
      const uint32_t kt = smem_u32(ring + st * 2 * kTileB);
      const uint32_t vt = kt + kTileB;

      // ---- scores: 2 row blocks of 16 keys x 4 k-steps of 32 channels
      float sc[NT][2][2];  // [nt][rb][key g, key g + 8]
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        int sacc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sacc[nt][e] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int mat = lane >> 3;
          const int row = warp * 32 + rb * 16 + (mat & 1) * 8 + (lane & 7);
          uint32_t a[4];
          ldsm_x4(kt + swz(row, 2 * j + (mat >> 1)), a);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_s8(sacc[nt], a, bq[nt][j][0], bq[nt][j][1]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float lo = f0[nt] * static_cast<float>(sacc[nt][0]) + f1[nt] * static_cast<float>(sacc[nt][1]);
          float hi = f0[nt] * static_cast<float>(sacc[nt][2]) + f1[nt] * static_cast<float>(sacc[nt][3]);
          lo += __shfl_xor_sync(0xffffffffu, lo, 1);
          hi += __shfl_xor_sync(0xffffffffu, hi, 1);
          const int key = base + rb * 16 + g;
          sc[nt][rb][0] = key < lim && !w.key.padding(key) ? lo : -INFINITY;
          sc[nt][rb][1] = key + 8 < lim && !w.key.padding(key + 8) ? hi : -INFINITY;
        }
      }
      // ---- online softmax per row; p' digits of this lane's own two keys
      __syncwarp();  // the previous tile's digit reads are done
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float mt = fmaxf(fmaxf(sc[nt][0][0], sc[nt][0][1]), fmaxf(sc[nt][1][0], sc[nt][1][1]));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 4));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 8));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 16));
        const float m_new = fmaxf(m_run[nt], mt);
        float pr[2], pv[2];
        float pm = 0.0f;
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
          const float sown = (t4 & 1) ? sc[nt][rb][1] : sc[nt][rb][0];
          pr[rb] = sown == -INFINITY ? 0.0f : exp2f(sown - m_new);
          pv[rb] = pr[rb] * vsf[rb];
          pm = fmaxf(pm, pv[rb]);
        }
        pm = fmaxf(pm, __shfl_xor_sync(0xffffffffu, pm, 1));
        pm = fmaxf(pm, __shfl_xor_sync(0xffffffffu, pm, 4));
        pm = fmaxf(pm, __shfl_xor_sync(0xffffffffu, pm, 8));
        pm = fmaxf(pm, __shfl_xor_sync(0xffffffffu, pm, 16));
        const bool rescale = m_new > m_run[nt];
        const bool grow = pm > pmax[nt];
        if (__any_sync(0xffffffffu, rescale || grow)) {
          flush(nt, rescale || grow);
          if (rescale) {
            const float alpha = exp2f(m_run[nt] - m_new);  // 0 on the first tile
            l_run[nt] *= alpha;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int pi = 0; pi < 2; ++pi) {
                o_acc[nt][j][pi][0] *= alpha;
                o_acc[nt][j][pi][1] *= alpha;
              }
          }
          // The digits' scale is chosen afresh where the maximum moves as well: what the earlier
          // keys needed is 2^(m - m_new) of itself now, and a scale left at it would round the
          // new leader away where its V scale is much smaller.
          if (rescale || grow) pmax[nt] = 2.0f * pm;
        }
        m_run[nt] = m_new;
        // (a seen key's V scale that is no number would get lost in the digits: the sum carries it)
        l_run[nt] += __fmaf_rn(0.0f, vsf[0], pr[0]) + __fmaf_rn(0.0f, vsf[1], pr[1]);
        const float inv_ps = pmax[nt] > 0.0f ? kLimbMax / pmax[nt] : 0.0f;
        unsigned char* dst = my_limb + nt * 256;
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
          const int x = min(__float2int_rn(pv[rb] * inv_ps), static_cast<int>(kLimbMax));
          int la, lb, lc;
          limbs24(x, la, lb, lc);
          const int k = pv_k(rb * 16 + g + 8 * (t4 & 1));
          const int hh = t4 >> 1;
          dst[(4 * hh + 0) * 32 + k] = static_cast<unsigned char>(la);
          dst[(4 * hh + 1) * 32 + k] = static_cast<unsigned char>(lb);
          dst[(4 * hh + 2) * 32 + k] = static_cast<unsigned char>(lc);
        }
      }
      __syncwarp();
      // ---- P V: A = V^T (ldmatrix.trans + byte permute), B = p' digits
      uint32_t bp[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const unsigned char* src = my_limb + nt * 256 + g * 32;
        bp[nt][0] = *reinterpret_cast<const uint32_t*>(src + 4 * t4);
        bp[nt][1] = *reinterpret_cast<const uint32_t*>(src + 16 + 4 * t4);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t ae[4], ao[4];
#pragma unroll
        for (int th = 0; th < 2; ++th) {
          const int mat = lane >> 3;
          const int row = warp * 32 + th * 16 + (mat & 1) * 8 + (lane & 7);
          uint32_t r[4];
          ldsm_x4_t(vt + swz(row, 2 * j + (mat >> 1)), r);
          ae[2 * th + 0] = prmt(r[0], r[1], 0x6420u);
          ao[2 * th + 0] = prmt(r[0], r[1], 0x7531u);
          ae[2 * th + 1] = prmt(r[2], r[3], 0x6420u);
          ao[2 * th + 1] = prmt(r[2], r[3], 0x7531u);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_s8(acc[nt][j][0], ae, bp[nt][0], bp[nt][1]);
          mma_s8(acc[nt][j][1], ao, bp[nt][0], bp[nt][1]);
        }
      }
      // 32 keys x 128 x 128 add up to 2^19 a tile and digit: int32 holds 4096 tiles
      if (++since == 2048) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) flush(nt, true);
        since = 0;
      }
    }

    if (!ok) break;

    // ---- the 4 warps' states into one, per row
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      flush(nt, true);
      const int r = 2 * nt + (t4 >> 1);
      float l = l_run[nt];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      if (r < NR) {
        float* dst = wo + (warp * NR + r) * kD;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int pi = 0; pi < 2; ++pi)  // even lane: the row-g channel, odd lane: row g + 8
            dst[32 * j + 2 * g + pi + 16 * (t4 & 1)] = (t4 & 1) ? o_acc[nt][j][pi][1] : o_acc[nt][j][pi][0];
        if (g == 0 && (t4 & 1) == 0) wm[warp * NR + r] = make_float2(m_run[nt], l);
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      if (r >= rows) break;
      float M = -INFINITY, L = 0.0f, O = 0.0f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) M = fmaxf(M, wm[i * NR + r].x);
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const float2 ml = wm[i * NR + r];
        const float f = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - M);
        L += ml.y * f;
        O += wo[(i * NR + r) * kD + d] * f;
      }
      if (w.slot < 0) {
        const int u = r / p.nrep, h = w.kvh * p.nrep + r - u * p.nrep;
        const float y = L <= 0.0f ? 0.0f : O / L;  // (a NaN stays)
        char* dst = out_row(p, w.b, u, h);
        if (p.q_dt == HQ_DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(dst)[d] = __float2bfloat16_rn(y);
        else reinterpret_cast<__half*>(dst)[d] = __float2half_rn(y);
      } else {
        float* dst = part_row(p, w.slot, r);
        if (d == 0) *reinterpret_cast<float2*>(dst) = make_float2(M, L);
        dst[4 + d] = O;
      }
    }
    __syncthreads();  // q' of the next piece goes where the sums lie
  }
  if (!ok) {
    report_error(p.status, HQ_ERR_DEVICE_TIMEOUT);
    if (tid == 0)  // no copy is in flight when the block ends
      for (int i = done; i < issued; ++i) mbar_wait(&full[i % kStagesM], (i / kStagesM) & 1);
  }
  // launched beside the kernel before it: complete only after it
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Codes [B, Hkv, cap, 128] in boxes of `keys` keys, 128-byte swizzle, zeros past cap.
inline int encode_map(CUtensorMap* m, const int8_t* base, const Seg& s, int Hkv, int keys,
                      const Maps& maps) {
  auto enc = dec::encode_fn();
  if (!enc) return HQ_ERR_UNSUPPORTED;
  const int in = maps.inner;
  const cuuint64_t cap = s.cap, heads = maps.hm ? Hkv : 1, ss = s.ss, sh = maps.hm ? s.sh : s.ss;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(kD), in ? heads : cap, in ? cap : heads,
                              static_cast<cuuint64_t>(maps.bm ? s.nb : 1)};
  const cuuint64_t strides[3] = {in ? sh : ss, in ? ss : sh, static_cast<cuuint64_t>(maps.bm ? s.sb : s.ss)};
  const cuuint32_t n = keys;
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(kD), in ? 1u : n, in ? n : 1u, 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<int8_t*>(base), dims, strides, box,
                         es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? HQ_OK : HQ_ERR_INVALID_ARGUMENT;
}

template <int NR>
int launch_rows(const Params& p, const Maps& maps, int grid, cudaStream_t st) {
  using C = RCfg<NR>;
  static std::atomic<uint64_t> ready{0};
  auto kern = rows_kernel<NR>;
  const int rc = set_smem(kern, C::smem(kMaxEntries), ready);
  if (rc != HQ_OK) return rc;
  return launch_after(kern, dim3(grid), kThreads, C::smem(p.seg.nb), st, p, maps);
}

int rows_stream(const Params& p, int grid, cudaStream_t st) {
  Maps maps{};
  const Seg& s = p.seg;
  // (an extent of 1, or a stride of 0, is one copy for all)
  maps.hm = p.Hkv > 1 && s.sh != 0;
  maps.bm = s.nb > 1 && s.sb != 0;
  maps.inner = maps.hm && s.sh < s.ss;
  int rc = HQ_OK;
  if (s.cap > 0) {  // (an empty cache is never read)
    rc = encode_map(&maps.k, s.k, s, p.Hkv, kBN, maps);
    if (rc == HQ_OK) rc = encode_map(&maps.v, s.v, s, p.Hkv, kBN, maps);
    if (s.sinks > 0 && s.window < s.cap) {  // (else the keys are one run)
      if (rc == HQ_OK) rc = encode_map(&maps.k8, s.k, s, p.Hkv, 8, maps);
      if (rc == HQ_OK) rc = encode_map(&maps.v8, s.v, s, p.Hkv, 8, maps);
    }
  }
  if (rc != HQ_OK) return rc;
  const int rows = s.units * p.nrep;
  if (rows == 1) return launch_rows<1>(p, maps, grid, st);
  if (rows == 2) return launch_rows<2>(p, maps, grid, st);
  return launch_rows<4>(p, maps, grid, st);
}

}  // namespace rag
}  // namespace hq
