// Decode attention over a paged 4-bit cache (paged4.cuh), one new token per sequence, lengths on the
// device (sm_100a).
//
// All sequences, kv heads and tokens are one line of 64-token tiles; every warp takes an equal run of
// it, with an online softmax of its own.  Units (sequence, kv head, up to 4 NT query rows) that end
// inside one warp's run are written by it; the ends of the warps' runs are joined in the block, and
// what crosses a block's border leaves partial states (m, l, o) that join_kernel puts together, always
// in the order of the line.
//
// 64 sequences of 4096 to 8192 tokens, 8 kv heads of 2 rows: 108 us, 4.2 TB/s of cache.  No unit is full
// (issue slots 49 %, arithmetic units 44 %, the matrix units 24 %, DRAM 47 % at half that size): the 8 warps
// that an SM has registers for do not hide the latency of a tile's chain of products, reductions and
// transpositions, and 144 bytes a token and head are 256 codes to unpack, twice.  Both products are
// whole-number products on bytes (mma.sync m16n8k32, exact), the codes being the 16-row operand, since a
// word of 8 codes becomes bytes with two masks and a shift (matrix instructions that take their operands
// from shared memory would want those bytes written there first: three times the tile's traffic):
//   * Q K^T: q is a 22-bit whole number per channel (of the row's largest |q|: 2^-22 of it is lost) in
//     three base-256 digits, two columns and a third in a second product, and -8 sum(q) added for the
//     codes' offset; one product is one group of 32 channels, its scale joins in float32.
//   * P V: p times the token's group scale, relative to the row's largest such product of the tile, is a
//     16-bit whole number (2^-16 of that product is lost of each; against the largest p and the largest
//     scale, each by itself, the tile took 3 % less time, but a large scale without weight left the others
//     no bits) in two digits, transposed in registers by movmatrix; four tokens' bytes are turned with
//     permutes.  A tile's sums go into the float32 state with the tile's and the group's factor.
// (As bf16 products, 7 to 12 instructions a word and twice the products, 64 x 8192 tokens took 138 us.)
// Up to 4 rows a kv head share one pass over its codes, up to 8 another that takes 1.5 times as long; more rows
// take a pass for every 8 of them (64 x 8192 whole tokens, 8 kv heads: 2 and 4 rows 136 us, 8 rows 207, 16
// rows 392, 128 rows 2861).
// Copies: every warp has its own ring of stages filled by bulk copies, one per page, side and kind,
// issued by one lane each.
#include <algorithm>
#include <atomic>

#include "paged4.cuh"
#include "umma.cuh"

namespace hq {
int current_sm_count();

namespace p4 {

constexpr int kTile = 64;                 // tokens
constexpr int kSets = kTile / 8;
constexpr int kWhole = 1024;              // tokens that one block takes in one go
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
  float* part;                            // states of blocks' ends
  float* ends;                            // and of warps'
  int* cum;                               // for join_kernel: first tile of every sequence
  int grid;
  int by_unit;                            // a block per unit, nothing to join across blocks
  int* status;
};

template <int NT>
struct Cfg {
  // 64 x 8192 tokens: 9 to 12 warps, their registers spilled, took 10 to 19 % more time, tiles of 32 tokens 10 %
  static constexpr int kWarps = 8;
  static constexpr int kStages = 2;
  static constexpr int kRows = 4 * NT;
  static constexpr int kOffBar = kWarps * kStages * kStageB;
  static constexpr int kOffCum = kOffBar + 8 * kWarps * kStages;
  static constexpr int kState = kRows * kPartRow;
  static_assert(2 * kWarps <= 32 && kStages * kStageB >= 4 * kState && kStageB % 16 == 0, "ends of the warps' runs");
  static constexpr int smem(int B) { return kOffCum + 4 * (2 * B + 1); }
  static_assert(smem(kMaxSeqs) <= 232448, "one block per SM");
};

__device__ __forceinline__ int seq_len(const DecodeParams& p, int b) {
  return min(max(p.lens[b], 0), p.pg.max_pages << p.pg.page_log);
}
__device__ __forceinline__ int tiles_of(int len) { return max(1, (len + kTile - 1) / kTile); }

// d = a b + c in whole numbers, bytes of a (16 x 32) and b (32 x 8) signed or not.  (c is a product's
// result or zero: four other registers would be gathered for each product.)
#define HQ_MMA_BYTES(NAME, A, B)                                                                          \
  __device__ __forceinline__ void NAME(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,   \
                                       uint32_t b0, uint32_t b1, const int (&c)[4]) {                     \
    asm("mma.sync.aligned.m16n8k32.row.col.s32." A "." B ".s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "      \
        "{%8, %9}, {%10, %11, %12, %13};"                                                                 \
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])                                                  \
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3])); \
  }
HQ_MMA_BYTES(mma_u8s8, "u8", "s8")
HQ_MMA_BYTES(mma_u8u8, "u8", "u8")
HQ_MMA_BYTES(mma_s8s8, "s8", "s8")
HQ_MMA_BYTES(mma_s8u8, "s8", "u8")
#undef HQ_MMA_BYTES
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&x);
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3_abs(float a, float b, float c) {  // of the magnitudes; NaN if any is
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 half2_of(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// A place on the line of tiles: unit `idx` of sequence e, whose first tile is `first`.
struct Cursor {
  int line, end;
  int e, idx, first;
  int len, nt;
};
__device__ __forceinline__ void enter(Cursor& c, const int* lens, int e) {
  c.e = e;
  c.len = lens[e];
  c.nt = tiles_of(c.len);
}
// from the last tile of a unit to the next one's first; `per` units a sequence
__device__ __forceinline__ void next_unit(Cursor& c, const int* lens, int per) {
  c.first += c.nt;
  if (++c.idx == per) {
    c.idx = 0;
    enter(c, lens, c.e + 1);
  }
}
// the whole number that a row's largest |q| becomes: below 2^21, and its upper digit below 32
constexpr float kFixed = 2088960.0f;
// and that a tile's largest weight becomes (taken to 2^-8 of itself: 32640 at most, 64 x 8 of them below 2^24)
constexpr float kWeight = 32512.0f;
// largest weights below this (2^-110 of p = 1 under a scale of 1) are taken for none
constexpr float kNoWeight = 7.7037198e-34f;
__device__ constexpr int kZero[4] = {0, 0, 0, 0};

__device__ __forceinline__ uint32_t pack_pair(float a, float b, int dt) {
  if (dt == HQ_DTYPE_BF16) return pack_bf16(a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// (m, l, o) into the state (M, L, acc).  A state whose sums are no number has a maximum of -inf and
// passes them on.
__device__ __forceinline__ void join_state(float& M, float& L, float4& acc, float m, float l, const float4& o) {
  const float top = fmaxf(M, m);
  const float f0 = M == -INFINITY ? 0.0f : exp2f(M - top), f1 = m == -INFINITY ? 0.0f : exp2f(m - top);
  M = top;
  L = L * f0 + l * f1;
  acc.x = acc.x * f0 + o.x * f1;
  acc.y = acc.y * f0 + o.y * f1;
  acc.z = acc.z * f0 + o.z * f1;
  acc.w = acc.w * f0 + o.w * f1;
}
__device__ __forceinline__ void store_row(const DecodeParams& p, int q_dt, int b, int h, int d, float L, const float4& o) {
  const float inv = L <= 0.0f ? 0.0f : 1.0f / L;
  *reinterpret_cast<uint2*>(static_cast<char*>(p.out) + 2 * (b * p.os[0] + h * p.os[1] + d)) =
      make_uint2(pack_pair(o.x * inv, o.y * inv, q_dt), pack_pair(o.z * inv, o.w * inv, q_dt));
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
  // units that the warps' runs cut: one that began before and ends here (its state in global memory),
  // and the last (its state where the warp's ring was)
  __shared__ int ends[C::kWarps][2];
  auto end_state = [&](int x) {
    return x & 1 ? reinterpret_cast<float*>(smem + (x >> 1) * C::kStages * kStageB)
                 : p.ends + (static_cast<int64_t>(blockIdx.x) * C::kWarps + (x >> 1)) * C::kState;
  };
  int* lens = cum + p.B + 1;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (lane == 0)
    for (int i = 0; i < C::kStages; ++i) mbar_init(&full[i], 1);
  if (lane < 2) ends[warp][lane] = -1;
  fence_mbar_init();
  const int per = p.Hkv * p.n_rt;
  Cursor cur{};
  int run = 0;                            // tiles of a block
  if (p.by_unit) {
    cur.e = static_cast<int>(blockIdx.x / static_cast<uint32_t>(per));
    cur.idx = static_cast<int>(blockIdx.x) - cur.e * per;
    cur.len = seq_len(p, cur.e);
    cur.nt = tiles_of(cur.len);
    const int chunk = (cur.nt + C::kWarps - 1) / C::kWarps;
    cur.line = min(warp * chunk, cur.nt);
    cur.end = min(cur.line + chunk, cur.nt);
    __syncwarp();
  } else {
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
    // an equal run of the line for each block, and of that for each warp
    run = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
    const int chunk = (run + C::kWarps - 1) / C::kWarps;
    {
      const int64_t from = static_cast<int64_t>(blockIdx.x) * run, upto = min(from + run, static_cast<int64_t>(total));
      cur.line = static_cast<int>(min(from + warp * chunk, upto));
      cur.end = static_cast<int>(min(static_cast<int64_t>(cur.line) + chunk, upto));
    }
    if (cur.line < cur.end) {
      int lo = 0, hi = p.B - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cum[mid] <= cur.line) lo = mid; else hi = mid - 1;
      }
      enter(cur, lens, lo);
      cur.idx = static_cast<uint32_t>(cur.line - cum[lo]) / static_cast<uint32_t>(cur.nt);
      cur.first = cum[lo] + cur.idx * cur.nt;
    }
  }
  const bool any = cur.line < cur.end;

  // ---- the copies' cursor, up to kStages tiles ahead.  Lane 4 i + kind copies codes (kind 0: K, 1: V)
  // or scales (2: K, 3: V) of the tile's i-th page.  (Pages are no smaller than 16 tokens.)
  Cursor ahead = cur;
  const int kind = lane & 3, part = lane >> 2 & 3;
  const int here = min(p.pg.page, kTile);  // tokens of a page in a tile
  const int row_log = kind < 2 ? 6 : 3;    // bytes of a row
  static_assert(kRowB == 64 && kScaleB == 8, "row_log");
  const char* lane_base = kind == 0 ? reinterpret_cast<const char*>(p.pg.k) : kind == 1 ? reinterpret_cast<const char*>(p.pg.v)
                        : kind == 2 ? reinterpret_cast<const char*>(p.pg.ksc) : reinterpret_cast<const char*>(p.pg.vsc);
  const uint32_t page_b = static_cast<uint32_t>(kind < 2 ? p.pg.cp : 2 * p.pg.sp);
  const int64_t head_b = kind < 2 ? p.pg.ch : 2 * p.pg.sh;
  const bool mine = lane < 16 && part * here < kTile;
  const uint32_t to0 = smem_u32(ring) + (kind == 0 ? 0 : kind == 1 ? kOffV : kind == 2 ? kOffKs : kOffVs) + (part * here << row_log);
  const uint32_t bar0 = smem_u32(full);
  const char* unit_base = nullptr;
  const int* table = nullptr;
  int tok = 0, win = 0, ids = 0;          // ids: 32 page numbers from table entry `win` on
  int issued = 0, st_in = 0;
  auto load_ids = [&](int at) {
    win = at & ~31;
    ids = (win + lane) << p.pg.page_log < ahead.len ? table[win + lane] : -1;
  };
  auto open_unit = [&](int t) {
    const int kvh = p.n_rt == 1 ? ahead.idx : ahead.idx / p.n_rt;
    unit_base = lane_base + kvh * head_b;
    table = p.pg.tables + ahead.e * p.pg.tstride;
    tok = t * kTile;
    load_ids(tok >> p.pg.page_log);
  };
  if (any) open_unit(ahead.line - ahead.first);
  auto issue = [&]() {
    if (ahead.line >= ahead.end) return;
    const int pi = tok >> p.pg.page_log;
    if (pi >= win + 32) load_ids(pi);
    const int id = __shfl_sync(0xffffffffu, ids, pi - win + part);
    const bool need = mine && tok + part * here < ahead.len;
    const bool good = need && static_cast<uint32_t>(id) < static_cast<uint32_t>(p.pg.n_pages);
    const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, good)) * (here * (kRowB + kScaleB) / 2);  // 4 lanes a page
    const uint32_t bar = bar0 + 8 * st_in;
    if (lane == 0)
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
    if (good)
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                       to0 + st_in * kStageB),
                   "l"(unit_base + static_cast<uint64_t>(static_cast<uint32_t>(id)) * page_b + ((tok & (p.pg.page - 1)) << row_log)),
                   "r"(here << row_log), "r"(bar)
                   : "memory");
    if (need && !good) report_error(p.status, HQ_ERR_INVALID_ARGUMENT);
    ++issued;
    st_in = st_in + 1 == C::kStages ? 0 : st_in + 1;
    tok += kTile;
    if (++ahead.line == ahead.first + ahead.nt && ahead.line < ahead.end) {
      next_unit(ahead, lens, per);
      open_unit(0);
    }
  };
  __syncwarp();
#pragma unroll 1
  for (int i = 0; i < C::kStages; ++i) issue();

  // tokens of this lane's slots n8 and n8 + 8 of a block of 16 (Q K^T's rows, P's entries)
  const int e1 = n8 & 1, slot_tok = 4 * e1 + ((n8 >> 1) ^ e1);
  // V: rows n8 (and n8 + 8) are channels of chunk vj, half vh
  const int vj = n8 & 3, vh = n8 >> 2;
  const uint32_t vsel = vh ? 0x7362u : 0x5140u;  // (a.b0, b.b0, a.b1, b.b1) of half vh
  // K rows of slots: byte offset of chunk c4 of token slot_tok; V: chunk vj of tokens c4, 4 + (c4 ^ 1)
  const int k_off = slot_tok * kRowB + 16 * (c4 ^ (slot_tok & 2));
  const int va = c4, vb = 4 + (c4 ^ 1);
  const int va_off = kOffV + va * kRowB + 16 * (vj ^ (va & 2)), vb_off = kOffV + vb * kRowB + 16 * (vj ^ (vb & 2));

  int done = 0, st = 0;
  uint32_t phase = 0;
  bool ok = true;
#pragma unroll 1
  while (ok && cur.line < cur.end) {
    // ---- a piece: tiles t0 .. t1 - 1 of one unit
    const int t0 = cur.line - cur.first, t1 = min(cur.nt, t0 + cur.end - cur.line);
    const int kvh = p.n_rt == 1 ? cur.idx : cur.idx / p.n_rt;
    const int row0 = (cur.idx - kvh * p.n_rt) * C::kRows;
    const int b = cur.e, len = cur.len;
    const bool whole = t0 == 0 && t1 == cur.nt;
    // B fragments of q: columns 2 r, 2 r + 1 are the upper two digits of row 4 nt + r (a product for each
    // nt), 2 r + nt its lowest (one more); a lane's bytes are the channels 8 c4 + {0, 2, 4, 6} and
    // + {1, 3, 5, 7} of a group
    uint32_t bq[NT][4][2], bl[4][2] = {};
    int off[NT][4];                       // -8 sum(q) of row c4
    float qk[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row0 + 4 * nt + (n8 >> 1);
      const bool real = r < p.nrep;
      const char* row = static_cast<const char*>(p.q) + 2 * (b * p.qs[0] + (kvh * p.nrep + r) * p.qs[1] + 8 * c4);
      uint4 raw[4];
      float big = 0.0f;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        raw[g] = real ? *reinterpret_cast<const uint4*>(row + 64 * g) : make_uint4(0, 0, 0, 0);
        float f[8];
        if (q_dt == HQ_DTYPE_BF16) Vec16<HQ_DTYPE_BF16>::unpack(raw[g], f);
        else Vec16<HQ_DTYPE_F16>::unpack(raw[g], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) big = max_nan(big, fabsf(f[e]));
      }
      big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // (not below 2^-100, so that the step stays finite; a row that is no number gives scores that are none)
      const float fix = kFixed / fmaxf(big, 7.8886091e-31f);
      const float unit = big < INFINITY ? 1.0f / fix : NAN;
      qk[nt] = __shfl_sync(0xffffffffu, unit, 8 * c4) * p.qk_scale;  // of row c4: a lane that has its columns
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float f[8];
        if (q_dt == HQ_DTYPE_BF16) Vec16<HQ_DTYPE_BF16>::unpack(raw[g], f);
        else Vec16<HQ_DTYPE_F16>::unpack(raw[g], f);
        uint32_t top[2] = {0, 0}, low[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int x = __float2int_rn(f[e] * fix), y = (x + 128) >> 8, z = (y + 128) >> 8;
          const uint32_t d = (n8 & 1 ? y - 256 * z : z) & 0xff, d0 = (x - 256 * y) & 0xff;
          top[e & 1] |= d << (8 * (e >> 1));
          low[e & 1] |= d0 << (8 * (e >> 1));
        }
        bq[nt][g][0] = top[0];
        bq[nt][g][1] = top[1];
        if ((n8 & 1) == nt) {
          bl[g][0] = low[0];
          bl[g][1] = low[1];
        }
      }
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      constexpr uint32_t k8 = 0x08080808u;
      int w[4];
      mma_u8s8(w, k8, k8, k8, k8, bl[g][0], bl[g][1], kZero);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        int u[4];
        mma_u8s8(u, k8, k8, k8, k8, bq[nt][g][0], bq[nt][g][1], kZero);
        off[nt][g] = -((u[0] * 256 + u[1]) * 256 + w[nt]);
      }
    }
    float m_run[NT], l_run[NT], o[NT][4][2][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m_run[nt] = -INFINITY;
      l_run[nt] = 0.0f;
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int m = 0; m < 2; ++m)
          o[nt][g][m][0] = o[nt][g][m][1] = 0.0f;
    }

#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      ok = tc::wait_bar(&full[st], phase);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      ++done;
      const unsigned char* s = ring + st * kStageB;
      if (++st == C::kStages) {
        st = 0;
        phase ^= 1;
      }
      const int left = len - t * kTile;   // tokens of the tile that exist
      float sc[NT][kSets];                // tokens 8 i + slot_tok
#pragma unroll
      for (int blk = 0; blk < kSets / 2; ++blk) {
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
        for (int nt = 0; nt < NT; ++nt) sc[nt][2 * blk] = sc[nt][2 * blk + 1] = 0.0f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          constexpr uint32_t kLow = 0x0f0f0f0fu;
          const uint32_t x0 = a0[g] & kLow, x1 = (a0[g] >> 4) & kLow, y0 = a1[g] & kLow, y1 = (a1[g] >> 4) & kLow;
          int w[4];
          mma_u8s8(w, x0, y0, x1, y1, bl[g][0], bl[g][1], kZero);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            int u[4];
            mma_u8s8(u, x0, y0, x1, y1, bq[nt][g][0], bq[nt][g][1], kZero);
            // 32 x 8 x 2^21 is 2^29: whole numbers all the way
            sc[nt][2 * blk] = __fmaf_rn(s0[g], static_cast<float>((u[0] * 256 + u[1]) * 256 + (w[nt] + off[nt][g])), sc[nt][2 * blk]);
            sc[nt][2 * blk + 1] = __fmaf_rn(s1[g], static_cast<float>((u[2] * 256 + u[3]) * 256 + (w[2 + nt] + off[nt][g])), sc[nt][2 * blk + 1]);
          }
        }
        const int tk = blk * 16 + slot_tok;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          sc[nt][2 * blk] = tk < left ? sc[nt][2 * blk] * qk[nt] : -INFINITY;
          sc[nt][2 * blk + 1] = tk + 8 < left ? sc[nt][2 * blk + 1] * qk[nt] : -INFINITY;
        }
      }
      // ---- softmax of the tile, relative to its own maximum; f brings it to the running one
      float f[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float mt = sc[nt][0];
#pragma unroll
        for (int i = 1; i < kSets; ++i) mt = fmaxf(mt, sc[nt][i]);
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
            for (int m = 0; m < 2; ++m) {
              o[nt][g][m][0] *= alpha;
              o[nt][g][m][1] *= alpha;
            }
        }
        f[nt] = mt == -INFINITY ? 0.0f : ex2(mt - m_run[nt]);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kSets; ++i) {
          sc[nt][i] = sc[nt][i] == -INFINITY ? 0.0f : ex2(sc[nt][i] - mt);
          sum += sc[nt][i];
        }
        l_run[nt] = __fmaf_rn(f[nt], sum, l_run[nt]);
      }
      // ---- P V, two groups at a time: 2 gg in columns 2 r, 2 gg + 1 in 2 r + 1
#pragma unroll
      for (int gg = 0; gg < 2; ++gg) {
        // the tokens' V scales, and the rows' largest weights p x scale (bf16: to 2^-8 of themselves)
        uint32_t u[kSets];
        float big[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) big[nt][0] = big[nt][1] = 0.0f;
#pragma unroll
        for (int i = 0; i < kSets; i += 2) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int tk = 8 * (i + e) + slot_tok;
            u[i + e] = *reinterpret_cast<const uint32_t*>(s + kOffVs + tk * kScaleB + 4 * gg);
            if (tk >= left) u[i + e] = 0;   // what no token wrote may be anything
          }
          const float2 x = half2_of(u[i]), y = half2_of(u[i + 1]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            big[nt][0] = max3_abs(big[nt][0], sc[nt][i] * x.x, sc[nt][i + 1] * y.x);
            big[nt][1] = max3_abs(big[nt][1], sc[nt][i] * x.y, sc[nt][i + 1] * y.y);
          }
        }
        float2 top[NT], inv[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          __nv_bfloat162 both = __floats2bfloat162_rn(big[nt][0], big[nt][1]);
#pragma unroll
          for (int d = 4; d <= 16; d <<= 1) both = __hmax2_nan(both, __shfl_xor_sync(0xffffffffu, both, d));
          top[nt] = __bfloat1622float2(both);
          inv[nt].x = top[nt].x < kNoWeight ? 0.0f : kWeight * rcp(top[nt].x);
          inv[nt].y = top[nt].y < kNoWeight ? 0.0f : kWeight * rcp(top[nt].y);
        }
        // weights as whole numbers, then as operands: digits of 32 tokens each
        uint32_t hi[NT][kSets / 2], lo[NT][kSets / 2];
#pragma unroll
        for (int i = 0; i < kSets / 2; ++i) {
          const float2 x = half2_of(u[2 * i]), y = half2_of(u[2 * i + 1]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            constexpr float kRound = 12582912.0f;  // 1.5 x 2^23: the whole number in the low bits
            const uint32_t a = transpose8(prmt(__float_as_uint(__fmaf_rn(sc[nt][2 * i] * x.x, inv[nt].x, kRound)),
                                               __float_as_uint(__fmaf_rn(sc[nt][2 * i] * x.y, inv[nt].y, kRound)), 0x5410u));
            const uint32_t b2 = transpose8(prmt(__float_as_uint(__fmaf_rn(sc[nt][2 * i + 1] * y.x, inv[nt].x, kRound)),
                                                __float_as_uint(__fmaf_rn(sc[nt][2 * i + 1] * y.y, inv[nt].y, kRound)), 0x5410u));
            lo[nt][i] = prmt(a, b2, 0x6420u);
            hi[nt][i] = prmt(a, b2, 0x7531u);
          }
        }
        int ch[NT][4], cl[NT][4];         // the codes' offset
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          constexpr uint32_t kM8 = 0xf8f8f8f8u;
          mma_s8s8(ch[nt], kM8, kM8, kM8, kM8, hi[nt][0], hi[nt][1], kZero);
          mma_s8u8(cl[nt], kM8, kM8, kM8, kM8, lo[nt][0], lo[nt][1], kZero);
#pragma unroll
          for (int k = 1; k < kSets / 4; ++k) {
            mma_s8s8(ch[nt], kM8, kM8, kM8, kM8, hi[nt][2 * k], hi[nt][2 * k + 1], ch[nt]);
            mma_s8u8(cl[nt], kM8, kM8, kM8, kM8, lo[nt][2 * k], lo[nt][2 * k + 1], cl[nt]);
          }
        }
        // the groups' words of chunk vj of token slots 2 c4 and 2 c4 + 1, set by set: both groups' in one
        // load, where there are registers for them (7 x 2501 tokens 10 us against 12; 64 x 8192 2 % more)
        uint2 vw[2 * kSets];
        if constexpr (NT == 1) {
#pragma unroll
          for (int i = 0; i < kSets; ++i) {
            vw[2 * i] = *reinterpret_cast<const uint2*>(s + i * 8 * kRowB + va_off + 8 * gg);
            vw[2 * i + 1] = *reinterpret_cast<const uint2*>(s + i * 8 * kRowB + vb_off + 8 * gg);
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int g = 2 * gg + e;
          auto word = [&](int i) -> uint32_t {
            if constexpr (NT == 1) return e == 0 ? vw[i].x : vw[i].y;
            else return *reinterpret_cast<const uint32_t*>(s + (i >> 1) * 8 * kRowB + (i & 1 ? vb_off : va_off) + 4 * g);
          };
          int h[NT][2][4], q8[NT][2][4];
#pragma unroll
          for (int k = 0; k < kSets / 4; ++k) {
            uint32_t a[2][4];             // [channels 0, 1 / 2, 3][operand register]
#pragma unroll
            for (int y8 = 0; y8 < 2; ++y8) {
              const int w0 = 8 * k + 4 * y8;
              const uint32_t x = prmt(word(w0), word(w0 + 1), vsel), y = prmt(word(w0 + 2), word(w0 + 3), vsel);
              const uint32_t b0 = prmt(x, y, 0x5410u), b1 = prmt(x, y, 0x7632u);
              constexpr uint32_t kLow = 0x0f0f0f0fu;
              a[0][2 * y8] = b0 & kLow;
              a[0][2 * y8 + 1] = (b0 >> 4) & kLow;
              a[1][2 * y8] = b1 & kLow;
              a[1][2 * y8 + 1] = (b1 >> 4) & kLow;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int m = 0; m < 2; ++m) {
                mma_u8s8(h[nt][m], a[m][0], a[m][1], a[m][2], a[m][3], hi[nt][2 * k], hi[nt][2 * k + 1], k ? h[nt][m] : ch[nt]);
                mma_u8u8(q8[nt][m], a[m][0], a[m][1], a[m][2], a[m][3], lo[nt][2 * k], lo[nt][2 * k + 1], k ? q8[nt][m] : cl[nt]);
              }
          }
          // 64 x 8 x 32640 is below 2^24: exact in float32
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float w = f[nt] * ((e ? top[nt].y : top[nt].x) * (1.0f / kWeight));
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              o[nt][g][m][0] = __fmaf_rn(w, static_cast<float>(h[nt][m][e] * 256 + q8[nt][m][e]), o[nt][g][m][0]);
              o[nt][g][m][1] = __fmaf_rn(w, static_cast<float>(h[nt][m][2 + e] * 256 + q8[nt][m][2 + e]), o[nt][g][m][1]);
            }
          }
        }
      }
      __syncwarp();
      issue();
    }
    if (!ok) break;

    // ---- the piece's rows: lane (n8, c4) holds row 4 nt + c4, channels 32 g + 8 vj + 4 vh + 2 m, + 1
    const int ch = 8 * vj + 4 * vh;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      l_run[nt] += __shfl_xor_sync(0xffffffffu, l_run[nt], 4);
      l_run[nt] += __shfl_xor_sync(0xffffffffu, l_run[nt], 8);
      l_run[nt] += __shfl_xor_sync(0xffffffffu, l_run[nt], 16);
    }
    if (whole) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = row0 + 4 * nt + c4;
        if (r >= p.nrep) continue;
        const float inv = l_run[nt] <= 0.0f ? 0.0f : 1.0f / l_run[nt];  // (a NaN stays)
        char* dst = static_cast<char*>(p.out) + 2 * (b * p.os[0] + (kvh * p.nrep + r) * p.os[1] + ch);
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<uint2*>(dst + 64 * g) =
              make_uint2(pack_pair(o[nt][g][0][0] * inv, o[nt][g][0][1] * inv, q_dt),
                         pack_pair(o[nt][g][1][0] * inv, o[nt][g][1][1] * inv, q_dt));
      }
    } else {
      // the run's first or last unit (a third cannot be cut): to be joined with the other warps'
      const int x = 2 * warp + (cur.line + t1 - t0 == cur.end);
      if (lane == 0) ends[warp][x & 1] = cur.e * per + cur.idx;
      float* dst = end_state(x);
      __syncwarp();                       // (the last tile has been read by all lanes)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float* row = dst + (4 * nt + c4) * kPartRow;
        if (n8 == 0) *reinterpret_cast<float2*>(row) = make_float2(m_run[nt], l_run[nt]);
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4*>(row + 4 + 32 * g + ch) =
              make_float4(o[nt][g][0][0], o[nt][g][0][1], o[nt][g][1][0], o[nt][g][1][1]);
      }
    }
    cur.line += t1 - t0;
    if (t1 == cur.nt && cur.line < cur.end) next_unit(cur, lens, per);
  }
  if (!ok) {
    report_error(p.status, HQ_ERR_DEVICE_TIMEOUT);
    for (int i = done; i < issued; ++i) tc::wait_bar(&full[i % C::kStages], (i / C::kStages) & 1);
  }
  __syncthreads();

  // ---- the ends of the warps' runs: those of one unit are joined, in order, and written where they are
  // all of it, else left for join_kernel.  A warp per unit and row, a lane per end.
  {
    const int mine = lane < 2 * C::kWarps ? ends[lane >> 1][lane & 1] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, mine);
    uint32_t firsts = __ballot_sync(0xffffffffu, mine >= 0 && lane == __ffs(same) - 1);
    for (int task = 0; firsts; firsts &= firsts - 1) {
      const int at = __ffs(firsts) - 1;
      const int unit = __shfl_sync(0xffffffffu, mine, at);
      const uint32_t set = __shfl_sync(0xffffffffu, same, at);
      for (int row = 0; row < C::kRows; ++row, ++task) {
        if (task % C::kWarps != warp) continue;
        float m = -INFINITY, l = 0.0f;
        if (set >> lane & 1) {
          const float2 ml = *reinterpret_cast<const float2*>(end_state(lane) + row * kPartRow);
          m = ml.x;
          l = ml.y;
        }
        float M = m;
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
        const float f = m == -INFINITY ? 0.0f : exp2f(m - M);
        float L = l * f;                  // (a sum that is no number stays one)
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (uint32_t left = set; left; left &= left - 1) {
          const int x = __ffs(left) - 1;
          const float g = __shfl_sync(0xffffffffu, f, x);
          const float4 o = *reinterpret_cast<const float4*>(end_state(x) + row * kPartRow + 4 + 4 * lane);
          acc.x = __fmaf_rn(o.x, g, acc.x);
          acc.y = __fmaf_rn(o.y, g, acc.y);
          acc.z = __fmaf_rn(o.z, g, acc.z);
          acc.w = __fmaf_rn(o.w, g, acc.w);
        }
        const int e = unit / per, idx = unit - e * per, kvh = idx / p.n_rt, r = (idx - kvh * p.n_rt) * C::kRows + row;
        const int n = p.by_unit ? 1 : tiles_of(lens[e]), first = p.by_unit ? 0 : cum[e] + idx * n;
        if (!p.by_unit && first / run != (first + n - 1) / run) {
          float* dst = p.part + (static_cast<int64_t>(unit + static_cast<int>(blockIdx.x)) * C::kRows + row) * kPartRow;
          if (lane == 0) *reinterpret_cast<float2*>(dst) = make_float2(M, L);
          *reinterpret_cast<float4*>(dst + 4 + 4 * lane) = acc;
        } else if (r < p.nrep) {
          store_row(p, q_dt, e, kvh * p.nrep + r, 4 * lane, L, acc);
        }
      }
    }
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
  const int run = (p.cum[p.B] + p.grid - 1) / p.grid;
  const int nt = (p.cum[b + 1] - p.cum[b]) / per;
  const int first = p.cum[b] + idx * nt, w0 = first / run, w1 = (first + nt - 1) / run;
  if (w0 == w1) return;                   // written by its only block
  const float* at = p.part + (static_cast<int64_t>(b * per + idx + w0) * rows + hr - rt * rows) * kPartRow;
  const int64_t dist = static_cast<int64_t>(rows) * kPartRow;
  float M = -INFINITY, L = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int i = warp; i <= w1 - w0; i += kJoinWarps) {
    const float* x = at + i * dist;
    const float2 ml = *reinterpret_cast<const float2*>(x);
    join_state(M, L, acc, ml.x, ml.y, *reinterpret_cast<const float4*>(x + 4 + 4 * lane));
  }
  sum[warp][lane] = acc;
  if (lane == 0) sum[warp][32] = make_float4(M, L, 0.0f, 0.0f);
  __syncthreads();
  if (warp) return;
#pragma unroll
  for (int i = 1; i < kJoinWarps; ++i) {
    const float4 ml = sum[i][32];
    join_state(M, L, acc, ml.x, ml.y, sum[i][lane]);
  }
  store_row(p, q_dt, b, h, 4 * lane, L, acc);
}

// ---------------------------------------------------------------- host
struct DecodePlan {
  int nt, n_rt, grid, by_unit;
  size_t cum_bytes, part_bytes, bytes;
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
  // Few units with tables of up to kWhole tokens: a block per unit, 2 tiles a warp at most, and no second
  // launch (1 x 512 tokens 7.2 us against 8.9, 20 x 200 6.4 against 10.3; units for several rounds of
  // blocks better share the line: 64 x 512 26 us against 20).
  pl.by_unit = cap <= kWhole && units <= current_sm_count();
  if (pl.by_unit) {
    pl.grid = static_cast<int>(units);
    pl.bytes = 1;
    return true;
  }
  pl.grid = static_cast<int>(std::min<int64_t>(current_sm_count(), tiles));
  pl.cum_bytes = align256(sizeof(int) * (B + 1));
  pl.part_bytes = align256(sizeof(float) * static_cast<size_t>(units + pl.grid) * rows * kPartRow);
  pl.bytes = pl.cum_bytes + pl.part_bytes + sizeof(float) * static_cast<size_t>(pl.grid) * (pl.nt == 1 ? Cfg<1>::kWarps * Cfg<1>::kState : Cfg<2>::kWarps * Cfg<2>::kState);
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
  decode_kernel<NT><<<pl.grid, 32 * C::kWarps, C::smem(p.by_unit ? 0 : p.B), st>>>(p, q_dt);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.by_unit) return static_cast<int>(e);
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

extern "C" int hq_paged4_decode(const hq_paged4_decode_args* args) {
  if (!args) return HQ_ERR_INVALID_ARGUMENT;
  const hq_paged4_decode_args& a = *args;
  if (a.B < 0 || a.Hq <= 0 || a.Hkv <= 0) return HQ_ERR_INVALID_ARGUMENT;
  if (a.D != p4::kD || a.Hq % a.Hkv || (a.q_dtype != HQ_DTYPE_BF16 && a.q_dtype != HQ_DTYPE_F16)) return HQ_ERR_UNSUPPORTED;
  const int rc = p4::check_pages(a.k_codes, a.v_codes, a.k_scale, a.v_scale, a.code_strides, a.scale_strides, a.n_pages,
                                 a.page_size, a.tables, a.table_stride, a.max_pages, a.B, a.Hkv);
  if (rc != HQ_OK) return rc;
  if (a.B == 0) return HQ_OK;
  auto al = [](const void* x, uintptr_t n) { return reinterpret_cast<uintptr_t>(x) % n == 0; };
  if (!a.q || !a.out || !a.lens || !al(a.q, 16) || !al(a.out, 8) || a.q_strides[0] % 8 || a.q_strides[1] % 8 ||
      a.out_strides[0] % 4 || a.out_strides[1] % 4)
    return HQ_ERR_INVALID_ARGUMENT;
  p4::DecodePlan pl{};
  if (!p4::plan_decode(pl, a.B, a.Hkv, a.Hq / a.Hkv, int64_t(a.page_size) * a.max_pages) || int64_t(a.B) * a.Hq > 0x7fffffff)
    return HQ_ERR_UNSUPPORTED;
  if (!pl.by_unit && (!a.workspace || a.workspace_bytes < pl.bytes || !al(a.workspace, 256))) return HQ_ERR_WORKSPACE;
  // the output has rows of its own (but for q's: a unit's are read before they are written)
  const Rows out = packed_rows(a.out, a.B, a.Hq, a.out_strides), q = packed_rows(a.q, a.B, a.Hq, a.q_strides);
  if (rows_meet(out) || (!same_rows(out, q) && rows_meet(out, q))) return HQ_ERR_INVALID_ARGUMENT;
  p4::DecodeParams p{};
  p.pg = p4::make_pages(a.k_codes, a.v_codes, a.k_scale, a.v_scale, a.code_strides, a.scale_strides, a.n_pages, a.page_size,
                        a.tables, a.table_stride, a.max_pages);
  p.q = a.q;
  p.out = a.out;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = a.q_strides[i];
    p.os[i] = a.out_strides[i];
  }
  p.B = a.B;
  p.Hkv = a.Hkv;
  p.nrep = a.Hq / a.Hkv;
  p.n_rt = pl.n_rt;
  p.lens = a.lens;
  p.qk_scale = a.sm_scale * 1.4426950408889634f;
  if (!pl.by_unit) {
    p.cum = static_cast<int*>(a.workspace);
    p.part = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + pl.cum_bytes);
    p.ends = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + pl.cum_bytes + pl.part_bytes);
  }
  p.grid = pl.grid;
  p.by_unit = pl.by_unit;
  p.status = a.status;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a.stream);
  return pl.nt == 1 ? p4::launch_decode<1>(p, a.q_dtype, pl, st) : p4::launch_decode<2>(p, a.q_dtype, pl, st);
}
