// Attention over an int8 KV cache for batches whose sequences have lengths of their own
// (sm_100a): a sliding window with sink tokens for decode steps and prefill chunks, and
// decode over a prefix that a group of sequences shares.
//
//   o = sum_j softmax_j(q . k_j / sqrt(D)) v_j,   k_j[d] = code * k_scale[d],
//                                                  v_j[d] = code * v_scale[j]
//
// A query at position p sees key j when j <= p and (j > p - window or j < sinks); a query
// over a shared prefix sees all of it and all of its own sequence's tokens.
//
// Mathematics.  One pass over the keys with the running maximum and sum of a softmax, in
// base 2.  The K scales, the softmax scale and log2(e) are folded into q once per row (q' =
// q k_scale sm_scale log2 e, times a power of two that brings the bound max |q| max k_scale on it
// to [2^13, 2^14), rounded to float16; for float16 models a second float16 holds what the first
// leaves over); the int8 K codes are exact in float16.  V's scale is split in two: v_scale_j
// = g_j 2^(E + e_j), where E belongs to the piece of work.  g_j goes into V's float16 tile
// (code g_j), e_j joins the exponent: with t_j = s_j + e_j and m a running maximum of t,
//   P_j = 2^(t_j - m) (float16),  O += P_j (code_j g_j),  l += P_j 2^-e_j (float32),
// and o = 2^E O / l for V scales of any size.  A tile whose V scales lie within 2^-4 .. 2^6
// of 2^E (nearly every one) has all e_j = 0, and costs nothing for them; the others look
// e_j up.  Float16 models always put the whole scale into e_j (not a whole number then), so
// that V stays exact.  m moves only when t grows by more than 14 (P <= 2^14), so O in tensor memory
// is rarely rescaled.  Roundings to float16, each off by 2^-11 of itself at most: q' (bf16 models),
// P (one float16; prefill_attn.cu keeps two parts of it), and for bf16 models g_j and code g_j, an
// eighth of the output's own half step.  Errors against float64 are 4 % (bf16) and 14 to 20 %
// (float16) above those of a float32 form rounded once; V scales below 2^-60 count as zero.
//
// Work.  Row r of a unit (kv head, sequence or group) is q head kvh * n_rep + r % n_rep of
// query r / n_rep; 128 rows sit on the 128 lanes of tensor memory.  A block has two groups of
// softmax warps, each with two S buffers of 64 keys and one O accumulator: for more than 128 rows
// the groups hold two row tiles that share every key tile and step through its halves, else (ALT)
// one row tile, and each group takes one half of every key tile with a softmax state of its own,
// joined at the end.  Keys that no row of the block can see are never read: a block's keys are
// numbered v = 0 .. nv - 1, the sinks first, then the window's run, and cut into tiles of 128.
// Decode kernels (STREAM) lay the tiles of all units in one line and give each block an equal run
// of it, whatever the lengths; a unit cut by a block border leaves partial states (m, l, O) that
// combine_kernel joins.  Prefill blocks take one row tile each (split over a few blocks when there
// are few).
//
// Roles of a block (one per SM, 20 warps): softmax warps (2 x 4, one thread per row; they also
// form q', 16 lanes a row), 4 warps that turn staged K codes into float16 with byte permutes and
// store them in the 128-byte-swizzled layout the MMA reads and 4 that do so for V, two that fill
// the staging rings with bulk copies, one that reads the V scales, and one that issues the
// tcgen05.mma products: S = Q K^T into tensor memory, O += P V with P read from tensor memory,
// where it overwrites the S it came from.  mbarriers order the roles; every wait is bounded.
//
// Measured (bf16, 16 q heads over 8 kv heads): causal chunks of 2 x 8192 under a window of 2048,
// 359 us = 675 TFLOP/s, 0.41 of the measured bf16 rate; 64 sequences over 32768 shared keys 48 us
// = 355 TFLOP/s, 1410 GB/s of codes.  What bounds it is the softmax warps' instruction latency: a
// step of 64 keys takes some 2000 cycles a warp, of which the exponentials alone need 512; tensor
// pipe 36 % busy, issue slots 58 %, exp2 unit 36 %; and a fifth of a block is its start and end.
// What it replaced, same sizes: one S buffer of 128 keys a group, so that the softmax waited for
// P V and the next S in turn, 436 us; operands of the products moved into uniform registers one by
// one under a branch (80 cycles a product), 487; a first-piece search in every role (cold code
// each time), 380; codes loaded into registers and converted from there, 4000 cycles a tile, since
// the proxy fence before each hand-over waited for the loads of the next tile.
#include <type_traits>

#include "ragged_common.cuh"
#include "umma.cuh"

namespace hq {
namespace rag {
using namespace tc;

// registers a thread after the split (softmax warps, the others)
constexpr int kSoftRegs = 120, kOtherRegs = 80;
constexpr int kSoft = 256;                // softmax threads: two groups of 128
constexpr int kConvThreads = 256;
constexpr int kBS = 64;                   // keys of a softmax step: half a tile
constexpr int kTileB = kBN * kD * 2;      // a float16 K, V or Q tile: 32 KB
constexpr int kStages = 2;                // K and V tiles in shared memory
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColO = 256;           // S buffers at columns 0 and 128

template <bool ALT, bool LO>
struct Cfg {
  static constexpr int kThreads = kSoft + kConvThreads + 128;
  static constexpr int kRowTiles = ALT ? 1 : 2;
  static constexpr int kParts = LO ? 2 : 1;
  // staging rings, one for K codes and one for V codes
  static constexpr int kSlots = 3;
  static constexpr int kSlotKeys = kRowTiles * kParts == 1 ? 64 : 32;
  static constexpr int kSlotB = kSlotKeys * kD;
  static constexpr int kLvSlots = LO ? 2 : 3;  // ring of what the tiles' V scales lead to
  static constexpr int kOffK = kRowTiles * kParts * kTileB;
  static constexpr int kOffV = kOffK + kStages * kTileB;
  static constexpr int kOffSlot = kOffV + kStages * kTileB;
  static constexpr int kOffE = kOffSlot + 2 * kSlots * kSlotB;     // [slot][e_j, 2^-e_j][128]
  static constexpr int kOffG = kOffE + kLvSlots * 2 * kBN * 4;     // [slot][128] g_j, float16 twice
  static constexpr int kOffInfo = kOffG + kLvSlots * kBN * 4;      // [slot]{any e_j, 2^E}
  static constexpr int kOffFac = kOffInfo + 16 * ((kLvSlots + 1) / 2);  // [row] undoes q's power of two
  static constexpr int kOffRow = kOffFac + kRowTiles * 128 * 4;     // ALT: [2][128] the groups' (m, l)
  static constexpr int kOffBar = kOffRow + (ALT ? 2 * kBN * 8 : 0);
  static constexpr int kBars = 1 + 4 * kStages + 4 * kSlots + 2 * kLvSlots + 4 + 4 + 4 + 1 + 1 + 1;
  static constexpr int kOffMisc = kOffBar + ((kBars * 8 + 15) & ~15);
  static constexpr int kOffCum = kOffMisc + 16;
  static_assert(kOffFac % 16 == 0 && kOffRow % 16 == 0 && kOffBar % 8 == 0, "vector accesses");
  static constexpr int smem(int entries) { return 1024 + kOffCum + 4 * (entries + 1); }
  static_assert(1024 + kOffCum + 4 * (kMaxEntries + 1) <= 232448, "one block per SM");
};

// ---------------------------------------------------------------- small helpers
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
      : "memory");
}
constexpr float kTinyScale = 8.6736174e-19f;  // 2^-60: V scales below count as zero
__device__ __forceinline__ float pow2i(int e) {  // 2^e, -126 <= e <= 127
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}
// four int8 codes -> two float16 pairs, exact: the biased byte under the exponent of 1024
__device__ __forceinline__ void codes_to_h2(uint32_t w, uint32_t& a, uint32_t& b) {
  const uint32_t u = w ^ 0x80808080u;
  const uint32_t k1152 = 0x64806480u;
  const uint32_t x = prmt(u, 0x64646464u, 0x4140u), y = prmt(u, 0x64646464u, 0x4342u);
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(a) : "r"(x), "r"(k1152));
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(b) : "r"(y), "r"(k1152));
}
__device__ __forceinline__ bool elect_one() {  // one lane of a converged warp
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}
// tcgen05.mma by the lane whose `lead` is set.  The whole warp runs the code around it, and a
// descriptor comes as its low word and a constant high word: so all operands stay in uniform
// registers (under a branch each product took six moves into them, 80 cycles).
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint32_t a_lo, uint32_t a_hi,
                                       uint32_t b_lo, uint32_t b_hi, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %7, 0;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], a, b, %6, p;\n\t}\n" ::"r"(lead),
      "r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(id), "r"(acc));
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b_lo,
                                       uint32_t b_hi, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\tsetp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 b, {%3, %4};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], b, %5, p;\n\t}\n" ::"r"(lead),
      "r"(d), "r"(a), "r"(b_lo), "r"(b_hi), "r"(id), "r"(acc));
}
__device__ __forceinline__ void commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}\n" ::"r"(lead),
      "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// 32 or 64 columns of this thread's lane
__device__ __forceinline__ void tmem_cols(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
      "%29, %30, %31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_cols(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
      "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, "
      "%36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, "
      "%53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63"
      "}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]),
        "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]),
        "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]),
        "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]),
        "=r"(r[63])
      : "r"(taddr));
}
// Per-token int8 fake quantization of 8 values of a row with the largest |value| am, rounded back
// to the model dtype.
template <int DT>
__device__ __noinline__ uint4 fake_quant(uint4 x, float am) {
  const Quantizer qz = Quantizer::from_amax(am);
  float f[8];
  Vec16<DT>::unpack(x, f);
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float a = static_cast<float>(qz.code(f[2 * e])) * qz.scale;
    const float b = static_cast<float>(qz.code(f[2 * e + 1])) * qz.scale;
    w[e] = pack_pair(a, b, DT);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// ---------------------------------------------------------------- softmax of one row tile
struct RowLim {
  int hi, lo, vsk;  // key v is seen when v <= hi and (v >= lo or v < vsk)
  // bit e: key v0 + e is seen
  __device__ __forceinline__ uint32_t bits(int v0) const {
    const uint32_t upto = below(hi + 1 - v0);
    return upto & (~below(lo - v0) | below(vsk - v0));
  }
  __device__ __forceinline__ static uint32_t below(int n) {  // bits 0 .. n - 1
    return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
  }
};
// Code size decides here: a straight run of instructions that is not in the instruction cache
// costs about 10 cycles each, and the SM's schedulers hold some 12 KB each.  So the loops below
// stay rolled as far as registers allow, and what is rare is a call.

// t may exceed the running maximum by this: P <= 2^14, 2^16 is float16's end, and what float16
// rounds away of the smallest P (2^-25) is nothing beside the row's largest, 1 at least
constexpr float kSlack = 14.0f;
// O *= a
__device__ __noinline__ void rescale(uint32_t o_addr, float a) {
#pragma unroll 1
  for (int c = 0; c < 8; ++c) {
    uint32_t o[16];
    tmem_ld16(o_addr + 16 * c, o);
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * a);
    tmem_st16(o_addr + 16 * c, o);
  }
}
// The running maximum takes this step's largest t in, O and l are rescaled where it moves.
// pv_bar: the barrier of the step before, whose P V must be in O by then.  (Two barriers in turn:
// S of this step follows P V of the step before that one, so no wait that is skipped here can
// leave a parity behind.)
__device__ __forceinline__ void move_max(float mx, uint32_t o_addr, bool first, uint64_t* pv_bar,
                                         uint32_t pv_par, float& m, float& l, bool& ok) {
  const bool move = mx > m + kSlack || (m == -INFINITY && mx != -INFINITY);
  if (!__any_sync(0xffffffffu, move)) return;
  float a = 1.0f;
  if (move) {
    a = ex2_ftz(m - mx);
    m = mx;
    l *= a;
  }
  if (first) return;
  ok = wait_bar(pv_bar, pv_par);
  ok = __all_sync(0xffffffffu, ok);
  if (!ok) return;
  tc_fence_after();
  rescale(o_addr, a);
}

// One step of one row, 64 keys: the running maximum, then P = 2^(t - m) over S, and l.  CH: the
// scores held at a time.  All 64 in registers save the second read, 32 save half of the code, which
// runs cold in short blocks: 2 x 8192 rows took 381 us with 64 and 407 with 32, one prompt of 512
// 14.0 and 13.3, 33 sequences over three prefixes 43.9 and 40.3, so one row tile a block takes 32.
// EXP: t = s fac + e_j with e_j from ev[j] and 2^-e_j from ev[128 + j], else t = s fac.
// mask: some row of the warp does not see all of the keys.
template <bool EXP, int CH>
__device__ __forceinline__ void softmax_step(uint32_t s_addr, uint32_t o_addr, const float* ev,
                                             float fac, int v0, const RowLim& lim, bool mask,
                                             bool first, uint64_t* pv_bar, uint32_t pv_par,
                                             float& m, float& l, bool& ok) {
  uint32_t s[CH];
  auto scores = [&](int c) {  // t (EXP) or s, -inf where unseen
    tmem_cols(s_addr + c, s);
    if constexpr (EXP) {
#pragma unroll
      for (int e = 0; e < CH; e += 4) {
        const float4 e4 = *reinterpret_cast<const float4*>(ev + c + e);
        s[e] = __float_as_uint(__fmaf_rn(__uint_as_float(s[e]), fac, e4.x));
        s[e + 1] = __float_as_uint(__fmaf_rn(__uint_as_float(s[e + 1]), fac, e4.y));
        s[e + 2] = __float_as_uint(__fmaf_rn(__uint_as_float(s[e + 2]), fac, e4.z));
        s[e + 3] = __float_as_uint(__fmaf_rn(__uint_as_float(s[e + 3]), fac, e4.w));
      }
    }
    if (mask) {
#pragma unroll
      for (int h = 0; h < CH; h += 32) {
        const uint32_t seen = lim.bits(v0 + c + h);
#pragma unroll
        for (int e = 0; e < 32; ++e) s[h + e] = seen & (1u << e) ? s[h + e] : 0xff800000u;
      }
    }
  };
  float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
  for (int c = 0; c < kBS; c += CH) {
    scores(c);
#pragma unroll
    for (int e = 0; e < CH; e += 2)
      x[(e >> 1) & 3] = fmaxf(x[(e >> 1) & 3], fmaxf(__uint_as_float(s[e]), __uint_as_float(s[e + 1])));
  }
  float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  if constexpr (!EXP) mx *= fac;
  move_max(mx, o_addr, first, pv_bar, pv_par, m, l, ok);
  if (!ok) return;
  const float nb = m == -INFINITY ? 0.0f : -m;
  // (scalar: packed pairs cost more moves than they save)
  float ls[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
  for (int c = 0; c < kBS; c += CH) {
    if (CH < kBS) scores(c);
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < CH; e += 4) {
      float t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        t[i] = ex2_ftz(EXP ? __uint_as_float(s[e + i]) + nb : __fmaf_rn(__uint_as_float(s[e + i]), fac, nb));
      if constexpr (EXP) {
        const float4 r4 = *reinterpret_cast<const float4*>(ev + kBN + c + e);
        ls[0] = __fmaf_rn(t[0], r4.x, ls[0]);
        ls[1] = __fmaf_rn(t[1], r4.y, ls[1]);
        ls[2] = __fmaf_rn(t[2], r4.z, ls[2]);
        ls[3] = __fmaf_rn(t[3], r4.w, ls[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) ls[i] += t[i];
      }
      w[e / 2 % 8] = pack_h2(t[0], t[1]);
      w[e / 2 % 8 + 1] = pack_h2(t[2], t[3]);
      if (e % 16 == 12) tmem_st8(s_addr + (c + e - 12) / 2, w);  // over S columns that have been read
    }
  }
  l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
  tmem_wait_st();
}

// softmax_step<true> with less code, for the rare tiles of bf16 models with e_j.
__device__ __forceinline__ void softmax_step_any(uint32_t s_addr, uint32_t o_addr, const float* ev,
                                                 float fac, int v0, const RowLim& lim, bool first,
                                                 uint64_t* pv_bar, uint32_t pv_par,
                                                 float& m, float& l, bool& ok) {
  float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < kBS; c += 16) {
    const uint32_t seen = lim.bits(v0 + c);
    uint32_t s[16];
    tmem_ld16(s_addr + c, s);
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const float4 e4 = *reinterpret_cast<const float4*>(ev + c + e);
      const float t0 = __fmaf_rn(__uint_as_float(s[e]), fac, e4.x);
      const float t1 = __fmaf_rn(__uint_as_float(s[e + 1]), fac, e4.y);
      const float t2 = __fmaf_rn(__uint_as_float(s[e + 2]), fac, e4.z);
      const float t3 = __fmaf_rn(__uint_as_float(s[e + 3]), fac, e4.w);
      x0 = fmaxf(x0, fmaxf(seen & (1u << e) ? t0 : -INFINITY, seen & (2u << e) ? t1 : -INFINITY));
      x1 = fmaxf(x1, fmaxf(seen & (4u << e) ? t2 : -INFINITY, seen & (8u << e) ? t3 : -INFINITY));
    }
  }
  move_max(fmaxf(x0, x1), o_addr, first, pv_bar, pv_par, m, l, ok);
  if (!ok) return;
  const float nb = m == -INFINITY ? 0.0f : -m;
  float ls[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
  for (int c = 0; c < kBS; c += 16) {
    const uint32_t seen = lim.bits(v0 + c);
    uint32_t s[16], w[8];
    tmem_ld16(s_addr + c, s);
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const float4 e4 = *reinterpret_cast<const float4*>(ev + c + e);
      const float4 r4 = *reinterpret_cast<const float4*>(ev + kBN + c + e);
      float t[4] = {__fmaf_rn(__uint_as_float(s[e]), fac, e4.x + nb),
                    __fmaf_rn(__uint_as_float(s[e + 1]), fac, e4.y + nb),
                    __fmaf_rn(__uint_as_float(s[e + 2]), fac, e4.z + nb),
                    __fmaf_rn(__uint_as_float(s[e + 3]), fac, e4.w + nb)};
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = seen & (1u << (e + i)) ? ex2_ftz(t[i]) : 0.0f;
      ls[0] = __fmaf_rn(t[0], r4.x, ls[0]);
      ls[1] = __fmaf_rn(t[1], r4.y, ls[1]);
      ls[2] = __fmaf_rn(t[2], r4.z, ls[2]);
      ls[3] = __fmaf_rn(t[3], r4.w, ls[3]);
      w[e / 2] = pack_h2(t[0], t[1]);
      w[e / 2 + 1] = pack_h2(t[2], t[3]);
    }
    tmem_st8(s_addr + c / 2, w);  // over S columns that have been read
  }
  l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
  tmem_wait_st();
}

// ---------------------------------------------------------------- the kernel
template <bool ALT, bool LO, bool STREAM>
__global__ void __launch_bounds__(Cfg<ALT, LO>::kThreads, 1) ragged_kernel(const __grid_constant__ Params p) {
  using C = Cfg<ALT, LO>;
  constexpr int MT = 128 * C::kRowTiles;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  // (an offset, not a rounded address: the compiler keeps knowing that this is shared memory)
  unsigned char* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
  float* eb = reinterpret_cast<float*>(smem + C::kOffE);
  uint32_t* gb = reinterpret_cast<uint32_t*>(smem + C::kOffG);
  float2* info = reinterpret_cast<float2*>(smem + C::kOffInfo);
  float* facs = reinterpret_cast<float*>(smem + C::kOffFac);
  float2* rowb = reinterpret_cast<float2*>(smem + C::kOffRow);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* q_full = bars;
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* st_full = v_empty + kStages;
  uint64_t* st_empty = st_full + 2 * C::kSlots;  // [K, V][slot]
  uint64_t* lv_full = st_empty + 2 * C::kSlots;
  uint64_t* lv_empty = lv_full + C::kLvSlots;
  uint64_t* s_full = lv_empty + C::kLvSlots;  // [group][S buffer]
  uint64_t* p_ready = s_full + 4;
  uint64_t* pv_done = p_ready + 4;             // (of P V)
  uint64_t* o_empty = pv_done + 4;
  uint64_t* drain = o_empty + 1;
  uint64_t* soft_bar = drain + 1;         // the softmax warps among themselves
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  float* two_e = reinterpret_cast<float*>(smem + C::kOffMisc + 8);  // ALT: 2^E of the piece
  int* cum = reinterpret_cast<int*>(smem + C::kOffCum);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kMmaWarp = (kSoft + kConvThreads) / 32, kCopyWarp = kMmaWarp + 1;  // K; V scales; V
  // combine_kernel's blocks may be scheduled; they wait for this grid
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    if (lane == 0) {
      mbar_init(q_full, kSoft / 32);
      for (int i = 0; i < kStages; ++i) {
        mbar_init(&k_full[i], kConvThreads / 64);
        mbar_init(&k_empty[i], 1);
        mbar_init(&v_full[i], kConvThreads / 64);
        mbar_init(&v_empty[i], 1);
      }
      for (int i = 0; i < 2 * C::kSlots; ++i) {
        mbar_init(&st_full[i], 1);
        mbar_init(&st_empty[i], kConvThreads / 64);
      }
      for (int i = 0; i < C::kLvSlots; ++i) {
        mbar_init(&lv_full[i], 1);
        mbar_init(&lv_empty[i], 1);
      }
      for (int i = 0; i < 4; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_ready[i], 4);
        mbar_init(&pv_done[i], 1);
      }
      mbar_init(o_empty, kSoft / 32);
      mbar_init(drain, 1);
      mbar_init(soft_bar, kSoft / 32);
      fence_mbar_init();
    }
  }
  if constexpr (STREAM) build_cum<MT, 1>(p, cum, C::kThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // 0: a block allocates all columns
  const uint32_t q_base = smem_u32(smem), k_base = smem_u32(smem + C::kOffK),
                 v_base = smem_u32(smem + C::kOffV);
  Walk walk = walk_start<MT, STREAM, 1>(p, cum);
  auto next_piece = [&](Walk& k, Piece& to) { return walk_next<MT, STREAM, 1>(k, p, cum, to); };
  // the first piece, for all roles at once: a copy of this code in each would run cold in each
  Piece w{};
  const bool any = next_piece(walk, w);
  // the block's tiles one after the other, whatever the piece
  struct Cursor {
    Walk k;
    Piece w;
    int t;
  };
  auto next_tile = [&](Cursor& c) -> bool {
    if (++c.t < c.w.t1) return true;
    do {
      if (!next_piece(c.k, c.w)) return false;
    } while (c.w.t0 >= c.w.t1);
    c.t = c.w.t0;
    return true;
  };

  // (the shares' sum is what the block was launched with, 640 x 96: launch() checks it)
  if (warp >= kSoft / 32) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  if (warp < kSoft / 32) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    // ================= softmax: one thread per row (ALT: and group)
    const int grp = warp >> 2, lr = tid & 127, r = ALT ? lr : tid;  // row of its tile, of the piece
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_addr = 128 * grp + lane_base;
    const uint32_t o_addr = kColO + 128 * grp + lane_base;
    int pc = 0, gt0 = 0, cnt = 0;       // pieces, tiles of the block before this piece, own steps
    bool ok = true;
    unsigned char* q_tile = smem + (ALT ? 0 : grp) * C::kParts * kTileB;
    auto chunk = [&](int c) {  // 8 channels of the row
      return reinterpret_cast<uint4*>(q_tile + (c >> 3) * (kBN * 128) + sw128(lr, c & 7));
    };
    // the chunks this thread forms of q' and of the output: ALT: half a row each
    constexpr int kCh = ALT ? 8 : 16;
    const int ch0 = ALT ? 8 * grp : 0;
    // a barrier of the softmax warps whose wait is bounded, as all waits here are
    uint32_t syncs = 0;
    auto soft_sync = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(soft_bar);
      ok = wait_bar(soft_bar, syncs++ & 1) && ok;
      __syncwarp();
    };
    for (bool go = any; ok && go; go = next_piece(walk, w), ++pc) {
      const int n_tiles = w.t1 - w.t0;
      float m = -INFINITY, l = 0.0f, fac = 0.0f, vscale = 1.0f;
      const Seg& s = p.seg;
      const bool live = r < w.rows;
      const int u = (w.row0 + r) / p.nrep, h = w.kvh * p.nrep + (w.row0 + r) - u * p.nrep;
      const int wr0 = 32 * (ALT ? warp & 3 : warp);        // the warp's first row
      if (n_tiles > 0) {
        // ---- q' of kForm rows (those the warp stores in the end), 16 lanes a row.  The Q tile is
        // free: every S of the piece before has been seen.
        constexpr int DT = LO ? HQ_DTYPE_F16 : HQ_DTYPE_BF16, kForm = ALT ? 16 : 32;
        const int fr0 = ALT ? wr0 + 16 * grp : wr0, c = lane & 15, odd = lane >> 4;
        uint64_t from;  // of row fr0 + lane
        {
          const int rr = w.row0 + min(fr0 + (lane & (kForm - 1)), w.rows - 1), uu = rr / p.nrep;
          from = reinterpret_cast<uint64_t>(p.q) +
                 2 * (w.b * s.qsb + uu * s.qsu + (w.kvh * p.nrep + rr - uu * p.nrep) * p.qsh);
        }
        float k8[8], km = 0.0f;
        uint32_t kb[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          kb[e] = load_bits(s.ksc, w.b * s.kscb + w.kvh * s.ksch + (4 * lane + e) * s.kscd, p.s_dt);
        {
          constexpr int NX = kForm / 2;
          uint4 x[NX];
#pragma unroll
          for (int i = 0; i < NX; ++i) {
            const int k = 2 * i + odd;
            const uint64_t src = __shfl_sync(0xffffffffu, from, k);
            x[i] = fr0 + k < w.rows ? reinterpret_cast<const uint4*>(src)[c] : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float k = scale_of(kb[e], p.s_dt) * p.qk_scale;
            k8[e] = __shfl_sync(0xffffffffu, k, 2 * c);
            k8[4 + e] = __shfl_sync(0xffffffffu, k, 2 * c + 1);
            km = fmaxf(km, fabsf(k));
          }
#pragma unroll
          for (int o = 16; o >= 1; o >>= 1) km = fmaxf(km, __shfl_xor_sync(0xffffffffu, km, o));
          // the rows' largest |q|: straight code, whose shuffles overlap
          float am[NX];
#pragma unroll
          for (int i = 0; i < NX; ++i)
            am[i] = absmax_of_x2<DT>(absmax_x2<DT>(absmax_x2<DT>(x[i].x, x[i].y), absmax_x2<DT>(x[i].z, x[i].w)));
#pragma unroll
          for (int o = 8; o >= 1; o >>= 1)
#pragma unroll
            for (int i = 0; i < NX; ++i) am[i] = fmaxf(am[i], __shfl_xor_sync(0xffffffffu, am[i], o));
#pragma unroll 1
          for (int i0 = 0; i0 < NX; i0 += 2) {  // (rolled, the rows move up: straight code would run cold)
            uint4 y[2] = {x[0], x[1]};
            const float a2[2] = {am[0], am[1]};
#pragma unroll
            for (int k = 0; k < NX - 2; ++k) {
              x[k] = x[k + 2];
              am[k] = am[k + 2];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (p.q_quant) y[i] = fake_quant<DT>(y[i], a2[i]);
              // 2^ex brings the bound max |q| max k_scale to [2^13, 2^14): the row's largest |q'|
              // may lie some powers of two below, of which float16 has 14 to spare
              const int ex = min(max(13 - (static_cast<int>(__float_as_uint(a2[i] * km) >> 23) - 127), -100), 100);
              const float mul = pow2i(ex);
              float f[8];
              Vec16<DT>::unpack(y[i], f);
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float y0 = f[2 * e] * k8[2 * e] * mul, y1 = f[2 * e + 1] * k8[2 * e + 1] * mul;
                hi[e] = pack_h2(y0, y1);
                if constexpr (LO) {
                  const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&hi[e]));
                  lo[e] = pack_h2(y0 - g.x, y1 - g.y);
                }
              }
              const int row = fr0 + 2 * (i0 + i) + odd;
              unsigned char* to = smem + (row >> 7) * C::kParts * kTileB + (c >> 3) * (kBN * 128) + sw128(row & 127, c & 7);
              *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
              if constexpr (LO) *reinterpret_cast<uint4*>(to + kTileB) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
              if (c == 0) facs[row] = pow2i(-ex);
            }
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        // the groups keep step from piece to piece: one without rows must not arrive for the
        // next piece in this one's phase, nor look at a tile two ahead of the other's
        ok = wait_bar(q_full, pc & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fac = facs[r];
      }
      const bool warp_live = wr0 < w.rows;
      const bool mine = ALT || w.rows > 128 * grp;          // this group has rows
      const int pos = w.key.pos0 + (s.step ? u : 0);
      const RowLim lim = {live ? pos - w.key.sh : 1 << 30,
                          live ? pos - s.window + 1 - w.key.sh : 0,
                          w.key.sh > 0 ? w.key.ns : s.sinks};
      const int steps = !mine ? 0 : ALT ? n_tiles : 2 * n_tiles;
      for (int i = 0; ok && i < steps; ++i, ++cnt) {
        const int t = ALT ? i : i >> 1, half = ALT ? grp : i & 1;
        const int slot = (gt0 + t) % C::kLvSlots, buf = cnt & 1;
        if (ALT || half == 0) ok = wait_bar(&lv_full[slot], ((gt0 + t) / C::kLvSlots) & 1);
        ok = ok && wait_bar(&s_full[2 * grp + buf], (cnt >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (warp_live) {
          const float* ev = eb + slot * 2 * kBN + kBS * half;
          const int v0 = (w.t0 + t) * kBN + kBS * half;
          const float2 ti = info[slot];
          vscale = ti.y;
          const bool need = v0 + kBS - 1 > lim.hi || (v0 < lim.lo && v0 + kBS > lim.vsk && lim.lo > lim.vsk);
          const bool mask = __any_sync(0xffffffffu, need);
          uint64_t* pvb = &pv_done[2 * grp + (buf ^ 1)];
          const uint32_t pvp = ((cnt - 1) >> 1) & 1;
          if (!LO && ti.x != 0.0f)
            softmax_step_any(s_addr + kBS * buf, o_addr, ev, fac, v0, lim, i == 0, pvb, pvp, m, l, ok);
          else
            softmax_step<LO, ALT ? 32 : 64>(s_addr + kBS * buf, o_addr, ev, fac, v0, lim, mask, i == 0, pvb, pvp, m, l, ok);
        }
        if (!ok) break;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[2 * grp + buf]);
      }
      if (!ok) break;
      gt0 += n_tiles;
      // ---- the rows' results
      if (steps > 0) {
        ok = wait_bar(&pv_done[2 * grp + ((cnt - 1) & 1)], ((cnt - 1) >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      // (rows that saw nothing have l = 0 and give zeros, whatever their O holds; a NaN stays)
      bool has0 = steps > 0 && !(l <= 0.0f), has1 = false;
      float f0 = 1.0f, f1 = 0.0f;
      if constexpr (ALT) {  // both groups' states; each thread then takes half of the columns
        rowb[tid] = make_float2(m, l);
        if (tid == 0) *two_e = vscale;
        tc_fence_before();
        soft_sync();
        tc_fence_after();
        const float2 a = rowb[lr], b = rowb[kBN + lr];
        has0 = n_tiles > 0 && !(a.y <= 0.0f);
        has1 = n_tiles > 0 && !(b.y <= 0.0f);
        m = fmaxf(a.x, b.x);
        f0 = a.x == -INFINITY ? 0.0f : ex2_ftz(a.x - m);
        f1 = b.x == -INFINITY ? 0.0f : ex2_ftz(b.x - m);
        l = a.y * f0 + b.y * f1;
        vscale = *two_e;
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const bool have = live && (has0 || has1);
      const uint32_t o0 = ALT ? kColO + lane_base : o_addr, o1 = kColO + 128 + lane_base;
      if (warp_live && mine) {
        const float scale = w.slot < 0 ? (have ? vscale / l : 0.0f) : vscale;
        f0 = has0 ? f0 * scale : 0.0f;
        f1 = has1 ? f1 * scale : 0.0f;
        float* prt = part_row(p, w.slot < 0 ? 0 : w.slot, r);
        if (w.slot >= 0 && live && (!ALT || grp == 0))
          *reinterpret_cast<float2*>(prt) = make_float2(have ? m : -INFINITY, have ? l : 0.0f);
#pragma unroll 1
        for (int c = ch0; c < ch0 + kCh; c += 2) {
          uint32_t o[16];
          float y[16];
          tmem_ld16(o0 + 8 * c, o);
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] = has0 ? __uint_as_float(o[e]) * f0 : 0.0f;
          if constexpr (ALT) {
            tmem_ld16(o1 + 8 * c, o);
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] += has1 ? __uint_as_float(o[e]) * f1 : 0.0f;
          }
          if (w.slot < 0) {  // into the Q tile
            uint32_t z[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = pack_pair(y[2 * e], y[2 * e + 1], p.q_dt);
            *chunk(c) = make_uint4(z[0], z[1], z[2], z[3]);
            *chunk(c + 1) = make_uint4(z[4], z[5], z[6], z[7]);
          } else if (live) {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *reinterpret_cast<float4*>(prt + 4 + 8 * c + e) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
          }
        }
      }
      if (n_tiles > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_empty);
      }
      if (w.slot < 0) {  // the warp's rows out, 256 bytes at a time
        if (ALT) soft_sync(); else __syncwarp();
        const uint64_t dst = reinterpret_cast<uint64_t>(out_row(p, w.b, u, h));
        const int i0 = ALT ? 16 * grp : 0, i1 = min(ALT ? i0 + 16 : 32, w.rows - wr0);
#pragma unroll 2
        for (int i = i0; i < i1; ++i) {
          char* to = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, dst, i));
          const int c = lane >> 1;
          const unsigned char* from = q_tile + (c >> 3) * (kBN * 128) +
                                      sw128((wr0 + i) & 127, c & 7) + 8 * (lane & 1);
          *reinterpret_cast<uint2*>(to + 8 * lane) = *reinterpret_cast<const uint2*>(from);
        }
      }
    }
    if (!ok) report_error(p.status, HQ_ERR_DEVICE_TIMEOUT);
  } else if (warp < kMmaWarp) {
    // ================= staged codes -> float16 tiles
    // 4 warps turn K, 4 V: fewer waits for each, and V, which waits for the P V of two tiles
    // before, holds up no K
    const bool is_v = warp >= (kSoft + kConvThreads / 2) / 32;
    const int ct = (tid - kSoft) % (kConvThreads / 2);
    // 8 codes (one 16-byte chunk) of rows row + 8 i of a slot: 8 lanes store 8 different chunk
    // columns, and rows 8 apart have the same swizzle
    const int c8 = ct & 15, row = ct >> 4;
    const uint32_t at = static_cast<uint32_t>(c8 >> 3) * (kBN * 128) + sw128(row, c8 & 7);
    bool ok = true;
    auto turn = [&](auto v, uint64_t* full, uint64_t* empty, uint64_t* sfull, uint64_t* sempty,
                    unsigned char* tiles, const unsigned char* slots) {
      constexpr bool V = decltype(v)::value;
      constexpr int NI = C::kSlotKeys / 8;
      int sl = 0, gt = 0;
      uint32_t sl_par = 0;
      Cursor c{walk, w, w.t0 - 1};
      for (; ok && next_tile(c); ++gt) {
        const int st = gt % kStages, use = gt / kStages;
        if (use > 0) ok = wait_bar(&empty[st], (use - 1) & 1);
        if constexpr (V) ok = ok && wait_bar(&lv_full[gt % C::kLvSlots], (gt / C::kLvSlots) & 1);
        const uint32_t* g = gb + gt % C::kLvSlots * kBN;
        unsigned char* to = tiles + st * kTileB + at;
#pragma unroll 1
        for (int k0 = 0; ok && k0 < kBN; k0 += C::kSlotKeys) {
          ok = wait_bar(&sfull[sl], sl_par);
          if (!ok) break;
          const unsigned char* src = slots + sl * C::kSlotB + row * kD + 8 * c8;
#pragma unroll 1
          for (int i0 = 0; i0 < NI; i0 += 4) {  // (all of a slot at once: 5 % slower, more code)
            uint2 x[4];
            uint32_t g2[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              x[i] = *reinterpret_cast<const uint2*>(src + (i0 + i) * 8 * kD);
              if constexpr (V) g2[i] = g[k0 + row + 8 * (i0 + i)];  // V rows times their g
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint4 y;
              codes_to_h2(x[i].x, y.x, y.y);
              codes_to_h2(x[i].y, y.z, y.w);
              if constexpr (V) {
                asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(y.x) : "r"(y.x), "r"(g2[i]));
                asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(y.y) : "r"(y.y), "r"(g2[i]));
                asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(y.z) : "r"(y.z), "r"(g2[i]));
                asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(y.w) : "r"(y.w), "r"(g2[i]));
              }
              *reinterpret_cast<uint4*>(to + (k0 + 8 * (i0 + i)) * 128) = y;
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sempty[sl]);
          if (++sl == C::kSlots) {
            sl = 0;
            sl_par ^= 1;
          }
        }
        if (!ok) break;
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[st]);
      }
    };
    if (is_v)
      turn(std::true_type{}, v_full, v_empty, st_full + C::kSlots, st_empty + C::kSlots,
           smem + C::kOffV, smem + C::kOffSlot + C::kSlots * C::kSlotB);
    else
      turn(std::false_type{}, k_full, k_empty, st_full, st_empty, smem + C::kOffK, smem + C::kOffSlot);
    if (!ok) report_error(p.status, HQ_ERR_DEVICE_TIMEOUT);
  } else if (warp == kCopyWarp || warp == kCopyWarp + 2) {
    // ================= codes into the staging ring
    const int is_v = warp == kCopyWarp + 2;
    uint64_t* full = st_full + is_v * C::kSlots;
    uint64_t* empty = st_empty + is_v * C::kSlots;
    unsigned char* slots = smem + C::kOffSlot + is_v * C::kSlots * C::kSlotB;
    int sc = 0;
    bool ok = true;
    Cursor c{walk, w, w.t0 - 1};
    while (ok && next_tile(c)) {
      const Seg& s = p.seg;
      const int8_t* src = (is_v ? s.v : s.k) + c.w.b * s.sb + c.w.kvh * s.sh;
#pragma unroll 1
      for (int v0 = c.t * kBN; v0 < (c.t + 1) * kBN; v0 += C::kSlotKeys, ++sc) {
        const int sl = sc % C::kSlots, use = sc / C::kSlots;
        if (use > 0) ok = wait_bar(&empty[sl], (use - 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int n = min(max(c.w.key.nv - v0, 0), C::kSlotKeys);
        unsigned char* dst = slots + sl * C::kSlotB;
        if (lane == 0) mbar_arrive_expect_tx(&full[sl], n * kD);
        __syncwarp();
        if (s.ss == kD) {  // rows back to back: the sinks' run and the window's
          const int n0 = min(max(c.w.key.ns - v0, 0), n);
          if (lane == 0 && n0 > 0) bulk_g2s(dst, src + static_cast<int64_t>(v0) * kD, n0 * kD, &full[sl]);
          if (lane == 0 && n > n0)
            bulk_g2s(dst + n0 * kD, src + static_cast<int64_t>(v0 + n0 + c.w.key.sh) * kD,
                     (n - n0) * kD, &full[sl]);
        } else {
          for (int i = lane; i < n; i += 32) {
            const int v = v0 + i;
            const int64_t key = v < c.w.key.ns ? v : v + c.w.key.sh;
            bulk_g2s(dst + i * kD, src + key * s.ss, kD, &full[sl]);
          }
        }
      }
    }
    if (!ok) report_error(p.status, HQ_ERR_DEVICE_TIMEOUT);
    // no copy is in flight when the block ends
    for (int k = max(0, sc - C::kSlots); k < sc; ++k)
      if (!mbar_wait(&full[k % C::kSlots], (k / C::kSlots) & 1))
        report_error(p.status, HQ_ERR_DEVICE_TIMEOUT);
  } else if (warp == kCopyWarp + 1) {
    // ================= V scales into g_j and e_j, loaded a tile ahead.  A scale that is no
    // number goes into e_j alone, where the mask comes after it: V's tile stays finite, and rows
    // that do not see the key keep their sums.
    int gt = 0;
    bool ok = true;
    Cursor c{walk, w, w.t0 - 1};  // of the loads
    uint32_t next[4];
    const uint32_t minus_one = p.s_dt == HQ_DTYPE_F32 ? __float_as_uint(-1.0f) : 0xbc00u;
    auto load_next = [&]() -> bool {
      if (!next_tile(c)) return false;
      const Seg& s = p.seg;
      const int64_t vs0 = c.w.b * s.vscb + c.w.kvh * s.vsch;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int v = c.t * kBN + 32 * i + lane;
        const int64_t key = v < c.w.key.ns ? v : v + c.w.key.sh;
        next[i] = v < c.w.key.nv ? load_bits(s.vsc, vs0 + key * s.vscs, p.s_dt) : minus_one;
      }
      return true;
    };
    bool have = load_next();
    int E = 0;
    while (have) {
      float vs[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) vs[i] = scale_of(next[i], p.s_dt);
      const bool first = c.t == c.w.t0;
      have = load_next();
      const int use = gt / C::kLvSlots, slot = gt % C::kLvSlots;
      if (use > 0) ok = wait_bar(&lv_empty[slot], (use - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      float* ev = eb + slot * 2 * kBN;
      bool any = LO;
      if constexpr (LO) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool zero = vs[i] < kTinyScale;
          const float x = zero ? kTinyScale : vs[i];
          ev[32 * i + lane] = __log2f(x);
          ev[kBN + 32 * i + lane] = x == x ? __frcp_rn(x) : 1.0f;
          gb[slot * kBN + 32 * i + lane] = zero ? 0u : 0x3c003c00u;
        }
      } else {
        int ex[4];
        bool odd = false;
        int top = -1000;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ex[i] = vs[i] < kTinyScale ? -60 : static_cast<int>(__float_as_uint(vs[i]) >> 23 & 255) - 127;
          top = max(top, vs[i] < kTinyScale || !(vs[i] < INFINITY) ? -1000 : ex[i]);
        }
        if (first) {
          top = __reduce_max_sync(0xffffffffu, top);
          E = top == -1000 ? 0 : min(max(top, -100), 100);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ex[i] -= E;
          odd = odd || !(vs[i] < INFINITY) || (vs[i] >= 0.0f && (ex[i] < -4 || ex[i] > 6 || vs[i] < kTinyScale));
        }
        any = __any_sync(0xffffffffu, odd);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = any ? min(max(ex[i], -100), 100) : 0;
          const bool zero = vs[i] < kTinyScale || !(vs[i] < INFINITY);
          ev[32 * i + lane] = vs[i] < INFINITY ? static_cast<float>(e) : NAN;
          ev[kBN + 32 * i + lane] = pow2i(-e);
          // (two factors: the exponent of their product may leave float32's)
          const float gj = zero ? 0.0f : vs[i] * pow2i(-E) * pow2i(-e);
          gb[slot * kBN + 32 * i + lane] = pack_h2(gj, gj);
        }
      }
      if (lane == 0) info[slot] = make_float2(any ? 1.0f : 0.0f, pow2i(E));
      __syncwarp();
      if (lane == 0) mbar_arrive(&lv_full[slot]);
      ++gt;
    }
    if (!ok) report_error(p.status, HQ_ERR_DEVICE_TIMEOUT);
  } else if (warp == kMmaWarp) {
    // ================= tensor-core products, issued by one thread; the warp stays together,
    // so that descriptors and addresses live in uniform registers
    {
      const uint32_t lead = elect_one();
      constexpr uint32_t id_s = idesc<HQ_DTYPE_F16>(128, kBS, false);
      constexpr uint32_t id_o = idesc<HQ_DTYPE_F16>(128, 128, true);
      // descriptors: the high word does not depend on the address, whose low word counts 16 bytes
      // (no sum leaves its 14 bits)
      constexpr uint32_t k_hi = sdesc(0, 16, 1024) >> 32, v_hi = sdesc(0, kBN * 128, 1024) >> 32;
      const uint32_t q_lo = static_cast<uint32_t>(sdesc(q_base, 16, 1024));
      const uint32_t k_lo = static_cast<uint32_t>(sdesc(k_base, 16, 1024));
      const uint32_t v_lo = static_cast<uint32_t>(sdesc(v_base, kBN * 128, 1024));
      bool ok = true;
      int g0 = 0, pieces = 0;   // tiles of the block before this piece, pieces
      int n0 = 0, n1 = 0;       // steps before this piece of each group
      // Step i of a piece, for group m: tile i and half m (ALT), or half i & 1 of tile i / 2
      auto tile_of = [&](int i) { return g0 + (ALT ? i : i >> 1); };
      auto k_wait = [&](int i) {
        const int g = tile_of(i);
        if (ALT || !(i & 1)) ok = ok && wait_bar(&k_full[g % kStages], (g / kStages) & 1);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      };
      auto k_done = [&](int i) {  // after the last S product that reads the tile
        if (ALT || (i & 1)) commit(lead, &k_empty[tile_of(i) % kStages]);
      };
      auto qk = [&](auto group, int i) {  // S = Q K^T
        constexpr int m = decltype(group)::value;
        const int buf = ((m ? n1 : n0) + i) & 1, half = ALT ? m : i & 1;
        const uint32_t b = k_lo + ((tile_of(i) % kStages * kTileB + half * kBS * 128) >> 4);
        const uint32_t a = q_lo + ((ALT ? 0 : m) * C::kParts * kTileB >> 4);
#pragma unroll
        for (int part = 0; part < C::kParts; ++part)
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint32_t off = ((kk >> 2) * (kBN * 128) + (kk & 3) * 32) >> 4;
            mma_ss(lead, 128 * m + kBS * buf, a + (part * (kTileB >> 4) + off), k_hi, b + off, k_hi,
                   id_s, part + kk > 0);
          }
        commit(lead, &s_full[2 * m + buf]);
      };
      auto pv = [&](auto group, int i) {  // O += P V
        constexpr int m = decltype(group)::value;
        const int n = (m ? n1 : n0) + i, buf = n & 1, half = ALT ? m : i & 1;
        ok = wait_bar(&p_ready[2 * m + buf], (n >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        tc_fence_after();
        const uint32_t b = v_lo + ((tile_of(i) % kStages * kTileB + half * kBS * 128) >> 4);
#pragma unroll
        for (int kk = 0; kk < kBS / 16; ++kk)
          mma_ts(lead, kColO + 128 * m, 128 * m + kBS * buf + 8 * kk, b + (kk * 16 * 128 >> 4), v_hi,
                 id_o, kk > 0 ? 1 : i > 0);
        commit(lead, &pv_done[2 * m + buf]);
      };
      using G0 = std::integral_constant<int, 0>;
      using G1 = std::integral_constant<int, 1>;
      // (all of the tensor memory is this block's: its columns count from 0)
      if (tmem != 0) ok = false;
      for (bool go = any; ok && go; go = next_piece(walk, w)) {
        const int n_tiles = w.t1 - w.t0, steps = ALT ? n_tiles : 2 * n_tiles;
        if (n_tiles <= 0) continue;
        const bool two = ALT || w.rows > 128;
        // (a piece's q is made by the warps that wait for the last P V of the piece before)
        ok = wait_bar(q_full, pieces & 1);
        // S of the first two steps; from then on S of step i + 2 follows P V of step i, whose P
        // lies in the same columns: the products run in order
#pragma unroll 1
        for (int i = 0; ok && i < min(steps, 2); ++i) {
          k_wait(i);
          if (!ok) break;
          qk(G0{}, i);
          if (two) qk(G1{}, i);
          k_done(i);
        }
        if (pieces > 0) ok = ok && wait_bar(o_empty, (pieces - 1) & 1);
        ++pieces;
#pragma unroll 1
        for (int i = 0; ok && i < steps; ++i) {
          const int g = tile_of(i);
          if (ALT || !(i & 1)) ok = wait_bar(&v_full[g % kStages], (g / kStages) & 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          pv(G0{}, i);
          if (!ok) break;
          const bool more = i + 2 < steps;
          if (more) {
            k_wait(i + 2);
            if (!ok) break;
            qk(G0{}, i + 2);
          }
          if (two) {
            pv(G1{}, i);
            if (!ok) break;
            if (more) qk(G1{}, i + 2);
          }
          if (ALT || (i & 1)) {
            commit(lead, &v_empty[g % kStages]);
            commit(lead, &lv_empty[g % C::kLvSlots]);  // (its readers are done with the tile, too)
          }
          if (more) k_done(i + 2);
        }
        g0 += n_tiles;
        n0 += steps;
        n1 += two ? steps : 0;
      }
      if (!ok) report_error(p.status, HQ_ERR_DEVICE_TIMEOUT);
      // every product has completed before the tensor memory is released
      commit(lead, drain);
      if (!mbar_wait(drain, 0)) report_error(p.status, HQ_ERR_DEVICE_TIMEOUT);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemCols)
                 : "memory");
  }
  // launched beside the kernel before it: complete only after it
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---------------------------------------------------------------- launches
template <bool ALT, bool LO, bool STREAM>
int launch(const Params& p, dim3 grid, cudaStream_t st) {
  using C = Cfg<ALT, LO>;
  static std::atomic<uint64_t> ready{0};
  auto kern = ragged_kernel<ALT, LO, STREAM>;
  // an increase beyond the registers of the launch would wait for ever
  static const bool fits = [&] {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, kern) == cudaSuccess &&
           a.numRegs * C::kThreads >= kSoft * kSoftRegs + (C::kThreads - kSoft) * kOtherRegs;
  }();
  if (!fits) return HQ_ERR_UNSUPPORTED;
  const int rc = set_smem(kern, C::smem(STREAM ? kMaxEntries : 0), ready);
  if (rc != HQ_OK) return rc;
  return launch_after(kern, grid, C::kThreads, C::smem(STREAM ? p.seg.nb : 0), st, p);
}

template <bool STREAM>
int dispatch(const Params& p, int nm, dim3 grid, cudaStream_t st) {
  if (p.q_dt == HQ_DTYPE_F16) return launch<true, true, STREAM>(p, grid, st);
  if (nm == 1) return launch<true, false, STREAM>(p, grid, st);
  return launch<false, false, STREAM>(p, grid, st);
}

int tiles_stream(const Params& p, int nm, int grid, cudaStream_t st) {
  return dispatch<true>(p, nm, dim3(grid), st);
}
int tiles_prefill(const Params& p, int nm, int B, cudaStream_t st) {
  return dispatch<false>(p, nm, dim3(p.n_split, p.Hkv * p.n_rt, B), st);
}

}  // namespace rag
}  // namespace hq
