// Causal attention of packed sequences of different lengths, 16-bit Q, K and V, grouped heads
// (sm_100a):  o_i = sum_j softmax_j(sm_scale q_i . k_j) v_j  over the keys j that query i sees.
//
// Sequence b has queries cu_q[b] .. cu_q[b + 1] - 1 and keys cu_k[b] .. cu_k[b + 1] - 1, the queries
// standing at its last positions: query i of n sees keys j <= m - n + i (all m, without the mask).
//
// Work.  Row r of a unit (sequence, kv head) is q head kvh n_rep + r % n_rep of query r / n_rep; 128
// rows are the lanes of a tile in tensor memory, and a block takes two tiles, 256 rows, that share
// every K and V tile of 128 keys.  Where that leaves SMs idle the keys are split over several blocks,
// whose states (m, l, O) join_kernel puts together.  How many is one number for the whole call, from averages
// that the host has: one long past beside many short sequences keeps its keys in one piece (plan()).  Blocks
// start from the end of the packed order, so of one sequence the pieces with the most keys come first; of
// several that is so where the last are the longest (16 sequences of 256 to 4096 tokens: 406 us in rising
// order, 407 to 419 in falling).  Every block looks for its sequence through all starts, 32 at a time: 64 sequences of
// one token 23 us, 1024 of them 420.
//
// Roles of a block: softmax warps, 4 or 8 a row tile; one warp that issues the products; one that loads K
// and V by TMA; two that look over the V tiles of masked steps.  S = Q K^T goes to tensor memory; the
// softmax threads take it into registers and write P in 16 bits over it; O += P V reads P from there.
// While one tile is in its softmax the other's products run.  The running maximum moves only when it grows
// by more than 8 (P <= 2^8), so O is rarely rescaled; sums are float32.  P is rounded to the model's type
// (2^-8 of each weight in bf16, 2^-11 in float16: what the output itself is rounded by; in float16 also
// 2^-32 of the largest).
//
// 2 x 8192 tokens of 16 q heads and 8 kv heads, bf16: 530 to 540 us in a run of calls, at 990 W and 1.64 GHz
// (455 to 462, 1200 TFLOP/s, in a burst).  Neither unit is full (1 x 8192:
// tensor 57 %, exponentials 58 %, issue slots 37 %): a row tile's scores, softmax and products follow one
// another, and two tiles a block leave gaps where both wait.  (Two threads a row take 19 % more; a quarter of the
// exponentials as polynomials no change, half of them 12 % more.)
//
// A V row holding an infinity or NaN spoils the rows that see it and no others: 0 x NaN is NaN in the
// product, so on steps where some row does not see every key such rows are zeroed in shared memory
// and rows that see them get a NaN sum.  (K needs none of this: unseen scores are replaced.)
#include <algorithm>
#include <atomic>

#include "decode_common.cuh"
#include "rows.cuh"
#include "umma.cuh"

namespace hq {
int current_sm_count();

namespace pk {
using namespace tc;

constexpr int kD = 128;
constexpr int kBN = 128;                  // keys per tile
constexpr int kTileB = kBN * kD * 2;
constexpr int kPartRow = kD + 4;
constexpr int kCleanWarps = 2;
constexpr int kMaxSplit = 16;

// A block's row tiles: two, one block per SM; or one, two blocks per SM (short sequences and small
// calls, where a block's start and end count).
template <int NT>
struct Cfg {
  static constexpr int kRows = 128 * NT;
  // Softmax threads: one a row with 128 keys, or (one row tile, where nothing hides a step's length) two with
  // 64 each, which tell each other their maxima.  One tile: 64 sequences of up to 200 tokens take 9 % less time
  // with two than with one, one of 512 8 %.  Two tiles: 2 x 8192 19 % more with two.
  static constexpr int kH = NT == 1 ? 2 : 1, kKeys = 128 / kH;
  static_assert(NT * kH <= 2, "places for one pair of threads a row");
  static constexpr int kSoft = 128 * NT * kH, kThreads = kSoft + 128;
  // registers a thread after the split (softmax warps, the others) of 168 at launch; 0: no split
  static constexpr int kSoftRegs = NT == 2 ? 208 : 0, kOtherRegs = NT == 2 ? 88 : 0;
  static constexpr int kPCol = 64 / (3 - kH);           // P of a tile's keys 64 .. : behind those before, or over their S
  static constexpr int kStages = 2 * NT;                // K, V, ..
  static constexpr int kOffKv = NT * kTileB;            // behind the Q tiles
  static constexpr int kOffBar = kOffKv + kStages * kTileB;
  static constexpr int kFull = 0, kEmpty = kFull + kStages, kSFull = kEmpty + kStages, kPFull = kSFull + NT,
                       kOFull = kPFull + 2 * NT, kPair = kOFull + NT, kClean = kPair + 4, kDrain = kClean + 2, kQ = kDrain + 1, kBars = kQ + 1;
  static constexpr int kOffBad = kOffBar + (kBars * 8 + 15) / 16 * 16;  // [2][4] words of spoiled V rows
  static constexpr int kOffHalf = kOffBad + 32;          // [2][kH][128] what the threads of a row tell each other
  static constexpr int kOffMisc = kOffHalf + (kH == 2 ? 2048 : 0);
  static constexpr int kSmem = 1024 + kOffMisc + 48;
  static constexpr uint32_t kColO = 128 * NT;           // tensor memory: S tiles, then O tiles
  static constexpr uint32_t kCols = 256 * NT;
};

struct Params {
  const void* q;
  void* out;
  int64_t qs[2], os[2];
  const int* cu_q;
  const int* cu_k;
  int T, Tk, B, Hkv, nrep;
  int causal;
  float c;                                // sm_scale log2(e)
  int n_split, units;                     // units: an upper bound of (sequence, piece of its rows, kv head)
  int swap;                               // tensor maps: (channel, token, head) instead of (channel, head, token)
  int q_tma;                              // Q tiles by tensor map: n_rep divides 128
  int zero_rest;
  float* part;
  int* status;
};

__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}
// Products by the lane whose `lead` is set, the warp converged (operands stay in uniform registers).
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo,
                                       uint32_t b_hi, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %7, 0;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], a, b, %6, p;\n\t}\n" ::"r"(lead),
      "r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(id), "r"(acc));
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi,
                                       uint32_t id, uint32_t acc) {
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
__device__ __forceinline__ void tmem_ld128(uint32_t taddr, uint32_t (&r)[128]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x128.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63, "
      "%64, %65, %66, %67, %68, %69, %70, %71, %72, %73, %74, %75, %76, %77, %78, %79, "
      "%80, %81, %82, %83, %84, %85, %86, %87, %88, %89, %90, %91, %92, %93, %94, %95, "
      "%96, %97, %98, %99, %100, %101, %102, %103, %104, %105, %106, %107, %108, %109, %110, %111, "
      "%112, %113, %114, %115, %116, %117, %118, %119, %120, %121, %122, %123, %124, %125, %126, %127"
      "}, [%128];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]),
        "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]),
        "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]),
        "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]),
        "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]),
        "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]),
        "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]),
        "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]),
        "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ldw32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31"
      "}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_stw16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {"
      "%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16"
      "};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_stw32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {"
      "%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32"
      "};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_ldw16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15"
      "}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  tmem_ldw16(taddr, r);
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float (&v)[16]) {
  uint32_t r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(v[i]);
  tmem_stw16(taddr, r);
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == HQ_DTYPE_BF16) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&x);
  } else {
    const __half2 x = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&x);
  }
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// ---------------------------------------------------------------- what a block works on
struct Seq {
  int q0, nq, k0, nk;
};
__device__ __forceinline__ Seq seq_of(const Params& p, int b) {
  Seq s;
  s.q0 = min(max(p.cu_q[b], 0), p.T);
  s.nq = min(max(p.cu_q[b + 1], s.q0), p.T) - s.q0;
  s.k0 = min(max(p.cu_k[b], 0), p.Tk);
  s.nk = min(max(p.cu_k[b + 1], s.k0), p.Tk) - s.k0;
  return s;
}
__device__ __forceinline__ int blocks_of(const Params& p, int nq, int rows) {
  return static_cast<int>((static_cast<int64_t>(nq) * p.nrep + rows - 1) / rows);
}
// All lanes of a warp: the sequence that holds piece u of the line of all sequences' pieces of `rows`
// rows (b = B: behind the last), and the piece's place in it.
__device__ __forceinline__ void find_piece(const Params& p, int u, int rows, int& b, int& y, Seq& s) {
  const int lane = threadIdx.x & 31;
  int run = 0;
  b = p.B;
  y = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    Seq mine{};
    if (b0 + lane < p.B) mine = seq_of(p, b0 + lane);
    const int n = blocks_of(p, mine.nq, rows);
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += z;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, run + x > u);
    if (hit) {
      const int l = __ffs(hit) - 1;
      b = b0 + l;
      y = u - run - __shfl_sync(0xffffffffu, x - n, l);
      s.q0 = __shfl_sync(0xffffffffu, mine.q0, l);
      s.nq = __shfl_sync(0xffffffffu, mine.nq, l);
      s.k0 = __shfl_sync(0xffffffffu, mine.k0, l);
      s.nk = __shfl_sync(0xffffffffu, mine.nk, l);
      return;
    }
    run += __shfl_sync(0xffffffffu, x, 31);
  }
}
// keys that row r of a unit sees: 0 .. lim - 1
__device__ __forceinline__ int limit_of(const Params& p, const Seq& s, int r) {
  const int i = static_cast<uint32_t>(r) / static_cast<uint32_t>(p.nrep);
  return p.causal ? min(max(s.nk - s.nq + i + 1, 0), s.nk) : s.nk;
}

template <int DT, int NT>
__global__ void __launch_bounds__(Cfg<NT>::kThreads, 3 - NT)
    packed_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap km,
                  const __grid_constant__ CUtensorMap vm) {
  using C = Cfg<NT>;
  constexpr int kRows = C::kRows, kThreads = C::kThreads, kStages = C::kStages, kSoftWarps = C::kSoft / 32;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint32_t* bad = reinterpret_cast<uint32_t*>(smem + C::kOffBad);
  int* misc = reinterpret_cast<int*>(smem + C::kOffMisc);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // rows before the first sequence and behind the last
  if (p.zero_rest) {
    const int first = min(max(p.cu_q[0], 0), p.T), end = min(max(p.cu_q[p.B], first), p.T);
    for (int64_t i = blockIdx.x; i < p.T - (end - first); i += gridDim.x) {
      const int64_t row = i < first ? i : i + (end - first);
      for (int x = tid; x < p.Hkv * p.nrep * (kD / 8); x += kThreads)
        *reinterpret_cast<uint4*>(static_cast<char*>(p.out) + 2 * (row * p.os[0] + x / (kD / 8) * p.os[1] + x % (kD / 8) * 8)) =
            make_uint4(0, 0, 0, 0);
    }
  }
  if (warp == 0) {
    // from the end: the last pieces of a sequence have the most keys
    const int item = p.units - 1 - static_cast<int>(blockIdx.x) / p.n_split;
    int b, y;
    Seq s{};
    find_piece(p, item / p.Hkv, kRows, b, y, s);
    if (lane == 0) {
      misc[0] = b;
      misc[1] = y;
      misc[2] = s.q0;
      misc[3] = s.nq;
      misc[4] = s.k0;
      misc[5] = s.nk;
    }
  }
  if (tid == 32) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bar[C::kFull + i], 1);
      mbar_init(&bar[C::kEmpty + i], i & 1 ? 1 + kCleanWarps : 1);  // V stages: products, and the warps that look
    }
    for (int t = 0; t < NT; ++t) {
      mbar_init(&bar[C::kSFull + t], 1);
      mbar_init(&bar[C::kPFull + 2 * t], 4);
      mbar_init(&bar[C::kPFull + 2 * t + 1], 4);
      mbar_init(&bar[C::kOFull + t], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&bar[C::kPair + i], 2);
    for (int i = 0; i < 2; ++i) mbar_init(&bar[C::kClean + i], kCleanWarps);
    mbar_init(&bar[C::kDrain], 1);
    mbar_init(&bar[C::kQ], 1);
    fence_mbar_init();
  }
  __syncthreads();
  if (misc[0] >= p.B) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const int split = static_cast<int>(blockIdx.x) % p.n_split, item = p.units - 1 - static_cast<int>(blockIdx.x) / p.n_split;
  const int kvh = item % p.Hkv;
  const Seq s = {misc[2], misc[3], misc[4], misc[5]};
  const int row0 = misc[1] * kRows, rows = min(kRows, s.nq * p.nrep - row0);  // rows >= 1
  // key tiles of the two row tiles, and the block's share of them
  int nt[NT], all = 0;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int last = min(rows, 128 * (t + 1)) - 1;
    nt[t] = last >= 128 * t ? (limit_of(p, s, row0 + last) + kBN - 1) / kBN : 0;
    all = max(all, nt[t]);
  }
  const int j0 = static_cast<int>(static_cast<int64_t>(all) * split / p.n_split);
  const int j1 = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / p.n_split);
  // masked steps: those from jm on, past the keys that every row sees.  The two barriers that say that
  // their V is looked over take turns: each V stage has its own, which cannot run a phase ahead.
  const int jm = max(j0, limit_of(p, s, row0) / kBN);
  auto clean_bar = [&](int j) { return &bar[C::kClean + (j & 1)]; };
  auto clean_phase = [&](int j) { return static_cast<uint32_t>((j - jm) >> 1) & 1u; };
  const uint32_t base = smem_u32(smem);

  if (warp == kSoftWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&misc[8])), "r"(C::kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  auto box = [&](const CUtensorMap* map, unsigned char* to, int x, int y, int z, uint64_t* full) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(to)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(full))
        : "memory");
  };
  // K and V tiles, in turn
  const int copies = 2 * (j1 - j0);
  auto copy = [&](int n) {
    const int st = n % kStages;
    const int key = s.k0 + (j0 + (n >> 1)) * kBN;
    mbar_arrive_expect_tx(&bar[C::kFull + st], kTileB);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      box(n & 1 ? &vm : &km, smem + C::kOffKv + st * kTileB + h * (kBN * 128), 64 * h, p.swap ? key : kvh, p.swap ? kvh : key,
          &bar[C::kFull + st]);
  };
  if (warp == kSoftWarps + 1 && lane == 0) {
    if (p.q_tma && copies) {  // 128 / n_rep queries a tile, all heads of each: its rows in order
      const int tiles = (rows + 127) / 128;
      mbar_arrive_expect_tx(&bar[C::kQ], tiles * kTileB);
      for (int t = 0; t < tiles; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          box(&qm, smem + t * kTileB + h * (kBN * 128), 64 * h, kvh * p.nrep, s.q0 + (row0 + 128 * t) / p.nrep, &bar[C::kQ]);
    }
    for (int n = 0; n < min(copies, kStages); ++n) copy(n);
  }
  // Q, 16 lanes a row: K-major tiles of two 64-channel halves, 128-byte swizzle; rows past the last: zeros.
  // (By tensor map, where n_rep divides 128, a block starts up to 1.5 us earlier: 64 sequences of up to 200
  // tokens take 8 % less time, 2 x 8192 1 %.  Rows past the last are then whatever follows: no row sees another.)
  if (!p.q_tma) {
    constexpr int kEach = (kRows * 16 + kThreads - 1) / kThreads;
    static_assert(kThreads % 16 == 0, "a half-warp per row");
    uint4 v[kEach];
    const int c = tid & 15;
    // row r's query and head, stepped from one of this thread's rows to the next
    const uint32_t nrep = p.nrep, first = row0 + (tid >> 4);
    uint32_t i = first / nrep, h = first - i * nrep;
    const uint32_t di = kThreads / 16 / nrep, dh = kThreads / 16 - di * nrep;
    const char* q = static_cast<const char*>(p.q) + 2 * (s.q0 * p.qs[0] + static_cast<int64_t>(kvh) * p.nrep * p.qs[1] + 8 * c);
#pragma unroll
    for (int n = 0; n < kEach; ++n) {     // all loads in flight at once (rows past the last read the first)
      const bool real = (tid >> 4) + n * (kThreads / 16) < rows;
      v[n] = *reinterpret_cast<const uint4*>(q + (real ? 2 * (i * p.qs[0] + h * p.qs[1]) : 0));
      i += di;
      h += dh;
      if (h >= nrep) {
        h -= nrep;
        ++i;
      }
    }
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
      const int r = (tid >> 4) + n * (kThreads / 16);
      if (r >= rows) v[n] = make_uint4(0, 0, 0, 0);
      if (r < kRows) *reinterpret_cast<uint4*>(smem + (r >> 7) * kTileB + (c >> 3) * (kBN * 128) + sw128(r & 127, c & 7)) = v[n];
    }
  }
  fence_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = static_cast<uint32_t>(misc[8]);
  bool ok = true;

  if constexpr (C::kSoftRegs > 0) {
    if (warp >= kSoftWarps) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftRegs));
  }
  if (warp < kSoftWarps) {
    // ------------------------------------------------------------ softmax: kH threads a row, kKeys keys each
    constexpr int kH = C::kH, kKeys = C::kKeys, kO = kH == 1 ? 32 : 16;  // (O's columns at a time)
    const int t = warp / (4 * kH), hf = kH == 2 ? warp >> 2 & 1 : 0, lr = 32 * (warp & 3) + lane, r = 128 * t + lr;
    const int lim = limit_of(p, s, row0 + min(r, rows - 1));
    const uint32_t tile = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
    const uint32_t s_addr = tile + 128 * t + kKeys * hf, o_addr = tile + C::kColO + 128 * t + kKeys * hf;
    // the other thread's value for this one's.  The place written turns from one call to the next, and the
    // second next one's comes when both have read: a step's products wait for both threads.
    auto exchange = [&](float v, int n) {
      float* at = reinterpret_cast<float*>(smem + C::kOffHalf) + 256 * (n & 1) + lr;
      uint64_t* pair = &bar[C::kPair + (warp & 3)];
      at[128 * hf] = v;
      __syncwarp();
      if (lane == 0) mbar_arrive(pair);
      ok = wait_bar(pair, n & 1);
      return at[128 * (hf ^ 1)];
    };
    float m = -INFINITY, l = 0.0f;        // m: of the raw scores
    const int jt = min(j1, nt[t]);
#pragma unroll 1
    for (int j = j0; j < jt; ++j) {
      ok = wait_bar(&bar[C::kSFull + t], (j - j0) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const int left = lim - j * kBN - kKeys * hf;  // keys of this thread's that its row sees
      const bool masked = j >= jm && __any_sync(0xffffffffu, left < kKeys);
      bool spoiled = false;
      // the scores: all of them in registers, or (fewer of those a thread) 32 at a time, twice
      constexpr int kHold = kH == 1 ? 128 : 32;
      uint32_t x[kHold];
      auto load = [&](int c) {
        if constexpr (kHold == 128) tmem_ld128(s_addr, x);
        else tmem_ldw32(s_addr + 32 * c, x);
        if (masked) {
#pragma unroll
          for (int i = 0; i < kHold; ++i) x[i] = kHold * c + i < left ? x[i] : 0xff800000u;
        }
      };
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < kKeys / kHold; ++c) {
        load(c);
        float m0 = fmaxf(top, __uint_as_float(x[0])), m1 = __uint_as_float(x[1]);
#pragma unroll
        for (int i = 2; i < kHold - 2; i += 4) {
          m0 = max3(m0, __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
          m1 = max3(m1, __uint_as_float(x[i + 2]), __uint_as_float(x[i + 3]));
        }
        top = max3(fmaxf(m0, m1), __uint_as_float(x[kHold - 2]), __uint_as_float(x[kHold - 1]));
      }
      if constexpr (kH == 2) {
        top = fmaxf(top, exchange(top, j - j0));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      if (j == j0) {
        m = top;
      } else if (__any_sync(0xffffffffu, (top - m) * p.c > 8.0f || (m == -INFINITY && top > m))) {
        // (lanes that need it and those that do not: the factor is 1 for a maximum that stays)
        const float m_new = (top - m) * p.c > 8.0f || (m == -INFINITY && top > m) ? top : m;
        const float f = m_new == m ? 1.0f : ex2_ftz((m - m_new) * p.c);
        m = m_new;
        l *= f;
#pragma unroll 1
        for (int i = 0; i < kKeys / kO; ++i) {
          float o[kO];
          if constexpr (kO == 32) tmem_ld32(o_addr + 32 * i, o);
          else tmem_ld16(o_addr + 16 * i, o);
#pragma unroll
          for (int e = 0; e < kO; ++e) o[e] *= f;
          if constexpr (kO == 32) tmem_st32(o_addr + 32 * i, o);
          else tmem_st16(o_addr + 16 * i, o);
        }
        tmem_wait_st();
      }
      // float16's weights are 2^7 times as large (up to 2^15): what it takes from small ones is 2^-32, not 2^-25,
      // of the largest, which many small ones would make felt.  O and l have the factor alike.
      constexpr float kLift = DT == HQ_DTYPE_F16 ? 7.0f : 0.0f;
      const float mc = (m == -INFINITY ? 0.0f : m * p.c) - kLift;
      const F2 c2 = f2_make(p.c, p.c), n2 = f2_make(-mc, -mc);
      F2 sum = f2_make(0.0f, 0.0f), sum1 = sum;
      // weights, over scores of this thread's that are read no more: those of the tile's keys 0 .. 63 at its
      // columns 0 .. 31, the others' from column kPCol on
      constexpr int kPiece = kHold == 32 ? 32 : 64;  // keys at a time
#pragma unroll
      for (int c = 0; c < kKeys / kPiece; ++c) {
        if constexpr (kHold == 32) load(c);
        constexpr int kAt = kHold == 32 ? 0 : kPiece;
        uint32_t w[kPiece / 2];
#pragma unroll
        for (int i = 0; i < kPiece / 2; ++i) {
          float a, e;
          f2_split(f2_fma(f2_make(__uint_as_float(x[kAt * c + 2 * i]), __uint_as_float(x[kAt * c + 2 * i + 1])), c2, n2), a, e);
          a = ex2_ftz(a);
          e = ex2_ftz(e);
          if (i & 1) sum = f2_add(sum, f2_make(a, e));
          else sum1 = f2_add(sum1, f2_make(a, e));
          w[i] = pack2<DT>(a, e);
        }
        if constexpr (kPiece == 64) tmem_stw32(s_addr + 32 * c, w);
        else tmem_stw16(s_addr + 16 * c, w);
        if (kPiece == 64 || c == 1) {     // 64 keys' weights are there
          tmem_wait_st();
          tc_fence_before();
          // spoiled V rows that this row sees (before the products may go on: they free V's stage, and with
          // it the barrier's next phase and the flags)
          if (c == kKeys / kPiece - 1 && j >= jm) {
            ok = wait_bar(clean_bar(j), clean_phase(j));
            const uint32_t* bits = bad + 4 * (j & 1) + 2 * hf;
#pragma unroll
            for (int i = 0; i < kKeys / 32; ++i) {
              const int n = min(max(left - 32 * i, 0), 32);
              spoiled |= (bits[i] & (n == 32 ? 0xffffffffu : (1u << n) - 1u)) != 0;
            }
          }
          ok = __all_sync(0xffffffffu, ok);
          if (ok && lane == 0) mbar_arrive(&bar[C::kPFull + 2 * t + (kH == 1 ? c : hf)]);
        }
      }
      if (!ok) break;
      float a, e;
      f2_split(f2_add(sum, sum1), a, e);
      l += a + e;
      if (spoiled) l = NAN;
    }
    // ---- the rows' results
    if (ok && jt > j0) {
      if constexpr (kH == 2) l += exchange(l, jt - j0);
      ok = ok && wait_bar(&bar[C::kOFull + t], 0);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    } else if (ok && p.q_tma && copies) {
      // a tile whose rows see no key here has awaited nothing: its Q, copied for the block's other tile's sake,
      // has to be there before zeros go over it
      ok = wait_bar(&bar[C::kQ], 0);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (ok && 128 * t + 32 * (warp & 3) < rows) {
      const bool live = r < rows, has = jt > j0 && !(l <= 0.0f);
      const float inv = has ? 1.0f / l : 0.0f;  // (a NaN stays)
      // a partial row's 4 channels c lie beside those of the other rows
      float4* prt = reinterpret_cast<float4*>(p.part + (static_cast<int64_t>(item) * p.n_split + split) * kRows * kPartRow);
      if (p.n_split > 1 && live && hf == 0)
        prt[r] = make_float4(has && m != -INFINITY ? m * p.c : -INFINITY, has ? l : 0.0f, 0.0f, 0.0f);
      // this tile's Q is read no more (its last product has been awaited, or its copy where there is none): its
      // rows' place, in halves of 128 bytes
      unsigned char* q_tile = smem + t * kTileB;
#pragma unroll 1
      for (int c = kKeys / kO * hf; c < kKeys / kO * (hf + 1); ++c) {
        float o[kO];
        if constexpr (kO == 32) tmem_ld32(tile + C::kColO + 128 * t + 32 * c, o);
        else tmem_ld16(tile + C::kColO + 128 * t + 16 * c, o);
        if (p.n_split > 1) {
          if (live)
#pragma unroll
            for (int e = 0; e < kO / 4; ++e)
              prt[(1 + kO / 4 * c + e) * kRows + r] =
                  has ? make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]) : make_float4(0, 0, 0, 0);
        } else {
#pragma unroll
          for (int e = 0; e < kO / 8; ++e) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (has)
              w = make_uint4(pack2<DT>(o[8 * e] * inv, o[8 * e + 1] * inv), pack2<DT>(o[8 * e + 2] * inv, o[8 * e + 3] * inv),
                             pack2<DT>(o[8 * e + 4] * inv, o[8 * e + 5] * inv), pack2<DT>(o[8 * e + 6] * inv, o[8 * e + 7] * inv));
            const int at = kO / 8 * c + e;  // of the row's 16 pieces
            *reinterpret_cast<uint4*>(q_tile + (at >> 3) * (kTileB / 2) + sw128(lr, at & 7)) = w;
          }
        }
      }
      __syncwarp();
      if (p.n_split == 1) {               // 16 / kH lanes a row
        constexpr uint32_t kLanes = 16 / kH, kStep = 32 / kLanes;
        const int c = lane % kLanes + 8 * hf;  // 16 bytes of the row
        const uint32_t nrep = p.nrep;
        int r2 = 32 * (warp & 3) + lane / kLanes;
        const uint32_t first = row0 + 128 * t + r2, i0 = first / nrep;
        uint32_t h = first - i0 * nrep;
        char* dst = static_cast<char*>(p.out) + 2 * ((s.q0 + static_cast<int64_t>(i0)) * p.os[0] + (kvh * p.nrep + static_cast<int64_t>(h)) * p.os[1] + 8 * c);
        const unsigned char* src = q_tile + (c >> 3) * (kTileB / 2);
        // kStep rows on: di queries and dh heads, or one query more where its heads end
        const uint32_t di = kStep / nrep, dh = kStep - di * nrep;
        const int64_t step = 2 * (di * p.os[0] + dh * p.os[1]), wrap = 2 * (p.os[0] - static_cast<int64_t>(nrep) * p.os[1]);
#pragma unroll 4
        for (int k = 0; k < 32 / static_cast<int>(kStep); ++k, r2 += kStep) {
          if (128 * t + r2 >= rows) break;
          *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src + sw128(r2, c & 7));
          dst += step;
          h += dh;
          if (h >= nrep) {
            h -= nrep;
            dst += wrap;
          }
        }
      }
    }
  } else if (warp == kSoftWarps) {
    // ------------------------------------------------------------ products
    const uint32_t lead = elect_one();
    constexpr uint32_t id_s = idesc<DT>(128, kBN, false), id_o = idesc<DT>(128, kD, true);
    constexpr uint32_t k_hi = sdesc(0, 16, 1024) >> 32, v_hi = sdesc(0, kBN * 128, 1024) >> 32;
    const uint32_t q_lo = static_cast<uint32_t>(sdesc(base, 16, 1024));
    const uint32_t k_lo = static_cast<uint32_t>(sdesc(base + C::kOffKv, 16, 1024));
    const uint32_t v_lo = static_cast<uint32_t>(sdesc(base + C::kOffKv, kBN * 128, 1024));
    auto score = [&](int t, int stage) {
      const uint32_t a = q_lo + (t * kTileB >> 4), k = k_lo + (stage * kTileB >> 4);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        const uint32_t off = ((kk >> 2) * (kBN * 128) + (kk & 3) * 32) >> 4;
        mma_ss(lead, tmem + 128 * t, a + off, k_hi, k + off, k_hi, id_s, kk > 0);
      }
      commit(lead, &bar[C::kSFull + t]);
    };
    if (j0 < j1) {
      ok = wait_bar(&bar[C::kFull], 0);
      if (p.q_tma) ok = ok && wait_bar(&bar[C::kQ], 0);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
          if (j0 < nt[t]) score(t, 0);
        commit(lead, &bar[C::kEmpty]);
      }
    }
#pragma unroll 1
    for (int j = j0; ok && j < j1; ++j) {
      const int n = j - j0, vi = 2 * n + 1, ki = 2 * n + 2;  // copies: V of this tile, K of the next
      const int vs = vi % kStages, ks = ki % kStages;
      ok = wait_bar(&bar[C::kFull + vs], (vi / kStages) & 1);
      if (j >= jm) ok = ok && wait_bar(clean_bar(j), clean_phase(j));
      if (j + 1 < j1) ok = ok && wait_bar(&bar[C::kFull + ks], (ki / kStages) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (j >= nt[t]) continue;
        const uint32_t v = v_lo + (vs * kTileB >> 4);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          ok = ok && wait_bar(&bar[C::kPFull + 2 * t + h], n & 1);
          if (C::kH == 2 && h == 0) ok = ok && wait_bar(&bar[C::kPFull + 2 * t + 1], n & 1);  // (both rescale O)
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
            mma_ts(lead, tmem + C::kColO + 128 * t, tmem + 128 * t + C::kPCol * h + 8 * (kk & 3), v + (kk * 16 * 128 >> 4), v_hi, id_o, n > 0 || kk > 0);
        }
        if (!ok) break;
        if (j + 1 < min(j1, nt[t])) score(t, ks);
        else commit(lead, &bar[C::kOFull + t]);
      }
      if (!ok) break;
      commit(lead, &bar[C::kEmpty + vs]);
      if (j + 1 < j1) commit(lead, &bar[C::kEmpty + ks]);
    }
    // no product is in flight when the block ends
    commit(lead, &bar[C::kDrain]);
    if (!wait_bar(&bar[C::kDrain], 0)) ok = false;
  } else if (warp == kSoftWarps + 1) {
    // ------------------------------------------------------------ copies
    int n = min(copies, kStages);
    if (lane == 0) {
      if (p.q_tma && copies) ok = wait_bar(&bar[C::kQ], 0);
      for (; ok && n < copies; ++n) {
        const int st = n % kStages;
        if (!(ok = wait_bar(&bar[C::kEmpty + st], (n / kStages - 1) & 1))) break;
        copy(n);
      }
      if (!ok)  // no copy is in flight when the block ends
        for (int i = max(0, n - kStages); i < n; ++i) wait_bar(&bar[C::kFull + i % kStages], (i / kStages) & 1);
    }
    ok = __all_sync(0xffffffffu, ok);
  } else {
    // ------------------------------------------------------------ V rows that hold no numbers, on masked steps
    const int g = warp - kSoftWarps - 2;
    constexpr uint32_t mask = DT == HQ_DTYPE_BF16 ? 0x7f807f80u : 0x7c007c00u, one = DT == HQ_DTYPE_BF16 ? 0x00800080u : 0x04000400u;
#pragma unroll 1
    for (int j = j0; j < j1; ++j) {
      const int vi = 2 * (j - j0) + 1, vs = vi % kStages;
      ok = wait_bar(&bar[C::kFull + vs], (vi / kStages) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (j < jm) {  // (every phase is waited for: a parity says nothing of phases further back)
        if (lane == 0) mbar_arrive(&bar[C::kEmpty + vs]);
        continue;
      }
      unsigned char* v = smem + C::kOffKv + vs * kTileB;
#pragma unroll 1
      for (int q = 0; q < 2; ++q) {
        const int row = 64 * g + 32 * q + lane;
        uint32_t seen = 0;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const uint4 x = *reinterpret_cast<const uint4*>(v + (c >> 3) * (kBN * 128) + row * 128 + (((c + lane) & 7) << 4));
          seen |= ((x.x & mask) + one) | ((x.y & mask) + one) | ((x.z & mask) + one) | ((x.w & mask) + one);
        }
        const bool broken = seen & 0x80008000u;
        if (broken)
          for (int c = 0; c < 16; ++c)
            *reinterpret_cast<uint4*>(v + (c >> 3) * (kBN * 128) + row * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
        const uint32_t word = __ballot_sync(0xffffffffu, broken);
        if (lane == 0) bad[4 * (j & 1) + 2 * g + q] = word;
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(clean_bar(j));
        mbar_arrive(&bar[C::kEmpty + vs]);
      }
    }
  }
  if (!ok && lane == 0) report_error(p.status, HQ_ERR_DEVICE_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == kSoftWarps) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kCols));
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Joins the pieces of a row tile, in order: block (piece of the line and kv head, 32 rows, 16 channels), a
// warp 8 rows, 4 lanes a row, 4 channels each: one round of loads.
template <int DT, int MOST>  // MOST: pieces at most (7 pieces with room for 16: 3 x 77 over 4022 22 us against 19)
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ Params p, int rows) {
  __shared__ int found[6];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int item = blockIdx.x, kvh = item % p.Hkv;
  if (warp == 0) {
    int b, y;
    Seq s{};
    find_piece(p, item / p.Hkv, rows, b, y, s);
    if (lane == 0) {
      found[0] = b;
      found[1] = y;
      found[2] = s.q0;
      found[3] = s.nq;
    }
  }
  __syncthreads();
  const int r = 32 * blockIdx.y + 8 * warp + (lane >> 2), row = found[1] * rows + r, cg = lane & 3;
  if (found[0] >= p.B || row >= found[3] * p.nrep) return;
  const float4* x = reinterpret_cast<const float4*>(p.part) + static_cast<int64_t>(item) * p.n_split * rows * (kPartRow / 4) + r;
  const int64_t step = static_cast<int64_t>(rows) * (kPartRow / 4);
  float f[MOST], l[MOST], M = -INFINITY, L = 0.0f;
  float4 o[MOST];
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    const float4 ml = i < p.n_split ? x[i * step] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
    f[i] = ml.x;
    l[i] = ml.y;
    if (i < p.n_split) o[i] = x[i * step + static_cast<int64_t>(1 + 4 * blockIdx.z + cg) * rows];
  }
#pragma unroll
  for (int i = 0; i < MOST; ++i) M = fmaxf(M, f[i]);
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    f[i] = f[i] == -INFINITY ? 0.0f : exp2f(f[i] - M);
    // (a piece whose sums are no number has a maximum of -inf and passes them on)
    L = __fmaf_rn(l[i], f[i], L);
  }
  const float inv = L <= 0.0f ? 0.0f : 1.0f / L;
  const int i = static_cast<uint32_t>(row) / static_cast<uint32_t>(p.nrep), h = kvh * p.nrep + row - i * p.nrep;
  char* dst = static_cast<char*>(p.out) + 2 * ((found[2] + static_cast<int64_t>(i)) * p.os[0] + h * p.os[1]);
  const int c = 4 * blockIdx.z + cg;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int k = 0; k < MOST; ++k)
    if (k < p.n_split) {
      acc.x = __fmaf_rn(o[k].x, f[k], acc.x);
      acc.y = __fmaf_rn(o[k].y, f[k], acc.y);
      acc.z = __fmaf_rn(o[k].z, f[k], acc.z);
      acc.w = __fmaf_rn(o[k].w, f[k], acc.w);
    }
  *reinterpret_cast<uint2*>(dst + 8 * c) = make_uint2(pack2<DT>(acc.x * inv, acc.y * inv), pack2<DT>(acc.z * inv, acc.w * inv));
}

// ---------------------------------------------------------------- host
struct Plan {
  int nt, units, n_split;
  size_t bytes;
};
inline bool plan(Plan& pl, int64_t T, int64_t Tk, int B, int Hkv, int nrep) {
  if (T * nrep > 0x3fffffff || Tk > 0x3fffffff) return false;
  const int sms = current_sm_count();
  // One row tile a block where sequences are short, in rows and in keys: 64 sequences of up to 200
  // tokens 45 us against 49 (32 of up to 300, 4 q heads a kv head, 85 and 85); with more of either, K and V
  // are better shared: 8 of 512 29 us against 32 (one of 512 14.9 and 14.4), one of 2048 38 against 40,
  // 2 x 8192 459 against 535, 3 x 77 queries over 4022 keys 19.5 against 21.5.
  pl.nt = T * nrep <= 512LL * B && Tk <= 1024LL * B ? 1 : 2;
  const int rows = 128 * pl.nt;
  // n rows are (n - 1) / rows + 1 pieces, rounded down; so are all sequences' at most
  const int64_t full = std::min<int64_t>(B, T), units = ((T * nrep - full) / rows + full) * Hkv;
  if (units * kMaxSplit > 0x7fffffff) return false;
  // With fewer blocks than fit the GPU each piece's keys go to several, as many as make the estimated time
  // least: 2 us a key tile of an average sequence; for more than one 3 us of a second launch (more than 8: 5.5), and
  // 0.15 ns a row and part for the states.  (Unsplit and split: 3 x 77 queries over 4022 keys 57 us and 19; 4 x 16 over 800 21
  // and 14; one of 1000 with 8 q heads over 2 kv heads 22 and 18; one of 512 14.7 and 16.1, 2 of 784 18.5 and
  // 20.3, which stay whole.  What averages miss: 16 queries over 32768 keys are split in 16 and take 39 us alone,
  // but 397 beside 16 sequences of one token, whose units leave the call unsplit.)
  const int64_t room = sms / std::max<int64_t>(units, 1);
  const int64_t tiles = (Tk + kBN * static_cast<int64_t>(B) - 1) / (kBN * static_cast<int64_t>(B));
  int64_t best = INT64_MAX;
  for (int64_t n = 1; n <= std::max<int64_t>(1, std::min<int64_t>({room, tiles, kMaxSplit})); ++n) {
    const int64_t ns = 2000 * ((tiles + n - 1) / n) + (n > 1 ? 3000 + 3 * T * nrep * Hkv * n / 20 : 0) + (n > 8 ? 2500 : 0);
    if (ns < best) {
      best = ns;
      pl.n_split = static_cast<int>(n);
    }
  }
  pl.units = static_cast<int>(units);
  pl.bytes = pl.n_split > 1 ? sizeof(float) * static_cast<size_t>(units) * pl.n_split * rows * kPartRow : 0;
  return true;
}

// [T, H, 128] in boxes of 64 channels, 128-byte swizzle, zeros past the end: of 128 tokens of a head, or of
// n_rep heads of 128 / n_rep tokens
inline int encode(CUtensorMap* m, const void* base, int dt, const int64_t st[2], int T, int H, int swap, int heads) {
  auto enc = dec::encode_fn();
  if (!enc) return HQ_ERR_UNSUPPORTED;
  const cuuint64_t ts = 2 * st[0], hs = H > 1 ? 2 * st[1] : (swap ? 2 * st[0] : 2 * kD);
  const cuuint64_t dims[3] = {kD, static_cast<cuuint64_t>(swap ? T : H), static_cast<cuuint64_t>(swap ? H : T)};
  const cuuint64_t strides[2] = {swap ? ts : hs, swap ? hs : ts};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(swap ? kBN : heads), static_cast<cuuint32_t>(swap ? 1 : kBN / heads)};
  const cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = enc(m, dt == HQ_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                         const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? HQ_OK : HQ_ERR_INVALID_ARGUMENT;
}

template <int DT, int NT>
int launch(const Params& p, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
  using C = Cfg<NT>;
  static std::atomic<uint64_t> ready{0};
  auto kern = packed_kernel<DT, NT>;
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = dev >= 0 && dev < 64 ? uint64_t(1) << dev : 0;
  if (!bit || !(ready.load(std::memory_order_acquire) & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return static_cast<int>(e);
    ready.fetch_or(bit, std::memory_order_acq_rel);
  }
  if (C::kSoftRegs > 0) {  // an increase beyond the registers of the launch would wait for ever
    static const bool fits = [&] {
      cudaFuncAttributes a;
      return cudaFuncGetAttributes(&a, kern) == cudaSuccess &&
             a.numRegs * C::kThreads >= C::kSoft * C::kSoftRegs + (C::kThreads - C::kSoft) * C::kOtherRegs;
    }();
    if (!fits) return HQ_ERR_UNSUPPORTED;
  }
  kern<<<p.units * p.n_split, C::kThreads, C::kSmem, st>>>(p, qm, km, vm);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.n_split == 1) return static_cast<int>(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.units, C::kRows / 32, kD / 16);
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = p.n_split <= 4   ? cudaLaunchKernelEx(&cfg, join_kernel<DT, 4>, p, C::kRows)
      : p.n_split <= 8 ? cudaLaunchKernelEx(&cfg, join_kernel<DT, 8>, p, C::kRows)
                       : cudaLaunchKernelEx(&cfg, join_kernel<DT, kMaxSplit>, p, C::kRows);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return static_cast<int>(e);
  }
  return HQ_OK;
}
template <int DT>
int launch(const Params& p, int nt, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
  return nt == 1 ? launch<DT, 1>(p, qm, km, vm, st) : launch<DT, 2>(p, qm, km, vm, st);
}

}  // namespace pk
}  // namespace hq

using namespace hq;

extern "C" size_t hq_packed_prefill_workspace_bytes(int T, int Tk, int B, int Hq, int Hkv, int D) {
  if (T <= 0 || Tk < 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D != pk::kD) return 0;
  pk::Plan pl{};
  return pk::plan(pl, T, Tk, B, Hkv, Hq / Hkv) ? std::max<size_t>(pl.bytes, 1) : 0;
}

extern "C" int hq_packed_prefill(const hq_packed_prefill_args* args) {
  if (!args) return HQ_ERR_INVALID_ARGUMENT;
  const hq_packed_prefill_args& a = *args;
  if (a.T < 0 || a.Tk < 0 || a.B < 0 || a.Hq <= 0 || a.Hkv <= 0 || !(a.sm_scale > 0.0f) || !(a.sm_scale < INFINITY))
    return HQ_ERR_INVALID_ARGUMENT;
  if (a.D != pk::kD || a.Hq % a.Hkv || (a.dtype != HQ_DTYPE_BF16 && a.dtype != HQ_DTYPE_F16)) return HQ_ERR_UNSUPPORTED;
  if (a.T == 0 || (a.B == 0 && !a.zero_rest)) return HQ_OK;
  auto al = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
  if (!a.q || !a.out || !a.cu_q || !a.cu_k || (a.Tk > 0 && (!a.k || !a.v)) || !al(a.q) || !al(a.k) || !al(a.v) || !al(a.out))
    return HQ_ERR_INVALID_ARGUMENT;
  const int64_t* in[4] = {a.q_strides, a.k_strides, a.v_strides, a.out_strides};
  for (const int64_t* s : in)
    if (s[0] % 8 || s[1] % 8 || s[0] < 0 || s[1] < 0) return HQ_ERR_INVALID_ARGUMENT;
  // TMA takes no stride of 0
  for (int i = 1; i < 3 && a.Tk > 0; ++i)
    if ((a.Tk > 1 && in[i][0] == 0) || (a.Hkv > 1 && in[i][1] == 0)) return HQ_ERR_INVALID_ARGUMENT;
  pk::Plan pl{};
  if (!pk::plan(pl, a.T, a.Tk, std::max(a.B, 1), a.Hkv, a.Hq / a.Hkv)) return HQ_ERR_UNSUPPORTED;
  if (pl.bytes && (!a.workspace || a.workspace_bytes < pl.bytes || !al(a.workspace))) return HQ_ERR_WORKSPACE;
  pk::Params p{};
  p.q = a.q;
  p.out = a.out;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = a.q_strides[i];
    p.os[i] = a.out_strides[i];
  }
  p.cu_q = a.cu_q;
  p.cu_k = a.cu_k;
  p.T = a.T;
  p.Tk = a.Tk;
  p.B = a.B;
  p.Hkv = a.Hkv;
  p.nrep = a.Hq / a.Hkv;
  p.causal = a.causal;
  p.c = a.sm_scale * 1.4426950408889634f;
  p.n_split = pl.n_split;
  p.units = pl.units;
  p.zero_rest = a.zero_rest;
  p.part = static_cast<float*>(a.workspace);
  p.status = a.status;
  // what is written has memory of its own (but for q's: a block reads no rows of others)
  const Rows out = packed_rows(a.out, a.T, a.Hq, a.out_strides), q = packed_rows(a.q, a.T, a.Hq, a.q_strides);
  if (rows_meet(out) || (!same_rows(out, q) && rows_meet(out, q)) || rows_meet(out, packed_rows(a.k, a.Tk, a.Hkv, a.k_strides)) ||
      rows_meet(out, packed_rows(a.v, a.Tk, a.Hkv, a.v_strides)))
    return HQ_ERR_INVALID_ARGUMENT;
  CUtensorMap qm{}, km{}, vm{};
  if (a.Tk > 0) {
    // strides in rising order, K's and V's alike
    p.swap = a.Hkv > 1 && a.k_strides[1] > a.k_strides[0];
    if (a.Hkv > 1 && (a.v_strides[1] > a.v_strides[0]) != (p.swap != 0)) return HQ_ERR_INVALID_ARGUMENT;
    const int64_t one = int64_t(a.Hkv) * pk::kD;
    const int64_t ks[2] = {a.Tk > 1 ? a.k_strides[0] : one, a.k_strides[1]}, vs[2] = {a.Tk > 1 ? a.v_strides[0] : one, a.v_strides[1]};
    int rc = pk::encode(&km, a.k, a.dtype, ks, a.Tk, a.Hkv, p.swap, 1);
    if (rc == HQ_OK) rc = pk::encode(&vm, a.v, a.dtype, vs, a.Tk, a.Hkv, p.swap, 1);
    if (rc != HQ_OK) return rc;
    // Q's rows in order come by tensor map: heads within tokens, no strides of 0
    const int64_t qs[2] = {a.T > 1 ? a.q_strides[0] : int64_t(a.Hq) * pk::kD, a.q_strides[1]};
    p.q_tma = 128 % p.nrep == 0 && qs[0] > 0 && (a.Hq == 1 || (qs[1] > 0 && qs[1] <= qs[0])) &&
              pk::encode(&qm, a.q, a.dtype, qs, a.T, a.Hq, 0, p.nrep) == HQ_OK;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a.stream);
  return a.dtype == HQ_DTYPE_BF16 ? pk::launch<HQ_DTYPE_BF16>(p, pl.nt, qm, km, vm, st)
                                  : pk::launch<HQ_DTYPE_F16>(p, pl.nt, qm, km, vm, st);
}
