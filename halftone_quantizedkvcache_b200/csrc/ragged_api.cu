// Plans, joining of partial states and entry points of the attention over int8 caches whose
// sequences have lengths of their own: sliding window with sinks (decode, prefill) and decode
// over a shared prefix.  The kernels are in ragged_attn.cu and ragged_rows.cu.
#include <algorithm>

#include "ragged_common.cuh"

namespace hq {
namespace rag {

// ---------------------------------------------------------------- joining the pieces
struct Source {
  Params p;
  int grid, mt;    // blocks that shared the line of tiles; rows per row tile
  int per_entry;   // sequences per entry (a prefix: those of its group)
};

// The partial rows of one output row in one source: first row, count, distance.
struct Run {
  const float* at;
  int n;
  int64_t step;
};
// STREAM: the blocks that hold tiles T0 .. T1 - 1 of a unit are T0 / per .. (T1 - 1) / per, and
// their pieces have consecutive slots.  n < 0: the row was written by the one block that held
// all of its tiles.
__device__ __forceinline__ Run stream_run(const Source& s, int b, int kvh, int hr) {
  const Params& p = s.p;
  const int e = b / s.per_entry, r = (b - e * s.per_entry) * p.nrep + hr;
  const int rt = r / s.mt, n_rt = row_tiles(p.seg.units * p.nrep, s.mt), idx = rt * p.Hkv + kvh;
  const int per = tiles_per_block(p, p.cum[p.seg.nb], s.grid);
  const int nt = (p.cum[e + 1] - p.cum[e]) / (p.Hkv * n_rt);
  if (nt == 0) return {nullptr, 0, 0};
  const int T0 = p.cum[e] + idx * nt, c0 = T0 / per, c1 = (T0 + nt - 1) / per;
  if (!p.merge_all && c0 == c1) return {nullptr, -1, 0};
  return {part_row(p, e * p.Hkv * n_rt + idx + c0, r - rt * s.mt), c1 - c0 + 1,
          static_cast<int64_t>(p.rows_cap) * kPartRow};
}
// Prefill: the n_split pieces of query u's row tile.
__device__ __forceinline__ Run split_run(const Source& s, int b, int u, int kvh, int hr) {
  const Params& p = s.p;
  const int r = u * p.nrep + hr, rt = r / s.mt;
  return {part_row(p, ((b * p.Hkv + kvh) * p.n_rt + rt) * p.n_split, r - rt * s.mt), p.n_split,
          static_cast<int64_t>(p.rows_cap) * kPartRow};
}

// One block per output row (b, u, h): warp w joins pieces w, w + 4, .., a lane 4 channels, under a
// maximum of its own, then warp 0 the warps' sums.  (One round of loads: finding the common maximum
// first took another.  A piece whose sums are no number has a maximum of -inf and passes them on.)
constexpr int kJoinWarps = 4;
template <int NSRC, bool STREAM>
__global__ void __launch_bounds__(32 * kJoinWarps) combine_kernel(const __grid_constant__ Source s0,
                                                                  const __grid_constant__ Source s1,
                                                                  int units) {
  __shared__ float4 sum[kJoinWarps][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Params& p = s0.p;
  const int h = blockIdx.y, b = STREAM ? blockIdx.x : blockIdx.x / units, u = blockIdx.x - b * units;
  const int kvh = h / p.nrep, hr = h - kvh * p.nrep;
  Run run[NSRC];
  if constexpr (STREAM) {
    run[0] = stream_run(s0, b, kvh, hr);
    if (run[0].n < 0) return;
    if constexpr (NSRC > 1) run[1] = stream_run(s1, b, kvh, hr);
  } else {
    const int nq = p.q_lens ? min(max(p.q_lens[b], 0), p.seg.units) : p.seg.units;
    if (u >= nq) return;
    run[0] = split_run(s0, b, u, kvh, hr);
  }
  float M = -INFINITY, L = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto join = [&](float m, float l, const float4& o) {
    const float top = fmaxf(M, m);
    const float f0 = M == -INFINITY ? 0.0f : exp2f(M - top), f1 = m == -INFINITY ? 0.0f : exp2f(m - top);
    M = top;
    L = L * f0 + l * f1;
    acc.x = acc.x * f0 + o.x * f1;
    acc.y = acc.y * f0 + o.y * f1;
    acc.z = acc.z * f0 + o.z * f1;
    acc.w = acc.w * f0 + o.w * f1;
  };
#pragma unroll
  for (int k = 0; k < NSRC; ++k)
#pragma unroll 4
    for (int i = warp; i < run[k].n; i += kJoinWarps) {
      const float* x = run[k].at + i * run[k].step;
      const float2 ml = *reinterpret_cast<const float2*>(x);
      join(ml.x, ml.y, *reinterpret_cast<const float4*>(x + 4 + 4 * lane));
    }
  sum[warp][lane] = acc;
  if (lane == 0) sum[warp][32] = make_float4(M, L, 0.0f, 0.0f);
  __syncthreads();
  if (warp) return;
#pragma unroll
  for (int i = 1; i < kJoinWarps; ++i) {
    const float4 ml = sum[i][32];
    join(ml.x, ml.y, sum[i][lane]);
  }
  const float inv = L <= 0.0f ? 0.0f : 1.0f / L;  // (a NaN stays)
  store4(out_row(p, b, u, h), p.q_dt, 4 * lane, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

template <int NSRC, bool STREAM>
int combine(const Source& s0, const Source& s1, int B, int units, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(B * units, s0.p.Hkv * s0.p.nrep);
  cfg.blockDim = dim3(32 * kJoinWarps);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, combine_kernel<NSRC, STREAM>, s0, s1, units);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return static_cast<int>(e);
  }
  return HQ_OK;
}

// ---------------------------------------------------------------- plans
inline size_t align256(size_t n) { return (n + 255) & ~size_t(255); }
inline bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Row tiles per block: two for more than 128 rows; float16 models (q' in two parts, whose
// second tile takes the shared memory of a second row tile) always one.
inline int tiles_of(int q_dt, int64_t rows) { return q_dt == HQ_DTYPE_F16 || rows <= 128 ? 1 : 2; }

// One line of tiles: `entries` sequences or groups with `rows` rows per kv head each.
struct Stream {
  bool few;          // ragged_rows.cu (two blocks per SM, no tensor memory)
  int nm, mt, grid, rows_cap;
  int64_t part_floats;
  size_t cum_bytes;
  size_t bytes() const { return cum_bytes + align256(sizeof(float) * static_cast<size_t>(part_floats)); }
};
inline bool plan_stream(Stream& pl, int q_dt, int Hkv, int entries, int64_t rows, int cap) {
  pl = Stream{};
  // Up to 4 rows (all it is built for): the int8 tensor-core kernel, whose work per key grows with
  // the rows and which needs no conversion of the codes; more: 128 rows at a time.  bf16, 8 kv heads,
  // at 1, 2, 3 and 4 rows: 64 sequences under a window of 4096, 94, 95, 123 and 125 us against 220 to
  // 221 for the other kernel; 8 sequences of up to 2048 tokens, 13, 14, 21 and 21 against 33 to 35;
  // one of 1024, 10, 10, 14 and 14 against 15 to 17.  Float16: the same, against 256, 37 and 17.
  pl.few = rows <= kMaxRows;
  pl.nm = pl.few ? 1 : tiles_of(q_dt, rows);
  pl.mt = 128 * pl.nm;
  const int64_t units = int64_t(entries) * Hkv * ((rows + pl.mt - 1) / pl.mt);
  const int64_t tiles = units * (cap / kBN + 1);
  if (tiles > (int64_t(1) << 30) || entries > kMaxEntries || rows > (1 << 24)) return false;
  pl.grid = static_cast<int>(std::min<int64_t>((pl.few ? 2 : 1) * int64_t(current_sm_count()),
                                               std::max<int64_t>(tiles, 1)));
  pl.rows_cap = static_cast<int>(std::min<int64_t>(rows, pl.mt));
  pl.part_floats = (units + pl.grid) * pl.rows_cap * kPartRow;
  pl.cum_bytes = align256(sizeof(int) * (entries + 1));
  return true;
}
inline void attach(Params& p, const Stream& pl, char* ws) {
  p.cum = reinterpret_cast<int*>(ws);
  p.part = reinterpret_cast<float*>(ws + pl.cum_bytes);
  p.rows_cap = pl.rows_cap;
  p.min_tiles = 1;
}
inline int run_stream(const Params& p, const Stream& pl, cudaStream_t st) {
  return pl.few ? rows_stream(p, pl.grid, st) : tiles_stream(p, pl.nm, pl.grid, st);
}

// Prefill plan: one block per row tile; with fewer blocks than SMs the keys of each row
// tile are split, down to two key tiles per block.
struct Prefill {
  int nm, n_rt, n_split, rows_cap;
  int64_t part_floats;
  size_t bytes() const { return align256(sizeof(float) * static_cast<size_t>(part_floats)); }
};
inline bool plan_prefill(Prefill& pl, int q_dt, int B, int Hkv, int nrep, int Sq, int cap, int window,
                         int sinks) {
  pl = Prefill{};
  const int64_t rows = int64_t(Sq) * nrep;
  if (rows > (1 << 30)) return false;
  pl.nm = tiles_of(q_dt, rows);
  // small grids keep one row tile per block
  if (pl.nm == 2 && int64_t(B) * Hkv * ((rows + 255) / 256) < current_sm_count()) pl.nm = 1;
  const int MT = 128 * pl.nm;
  pl.n_rt = static_cast<int>((rows + MT - 1) / MT);
  const int64_t units = int64_t(B) * Hkv * pl.n_rt;
  if (units * 64 > (int64_t(1) << 31) - 1 || int64_t(Hkv) * pl.n_rt > 65535) return false;
  const int64_t seen = std::min<int64_t>(cap, int64_t(window) + sinks + MT / nrep + 1);
  const int64_t nt = std::max<int64_t>(1, (seen + kBN - 1) / kBN);
  const int sms = current_sm_count();
  pl.n_split = static_cast<int>(std::min<int64_t>({std::max<int64_t>(1, sms / std::max<int64_t>(units, 1)),
                                                   std::max<int64_t>(1, nt / 2), 16}));
  pl.rows_cap = static_cast<int>(std::min<int64_t>(rows, MT));
  pl.part_floats = pl.n_split > 1 ? units * pl.n_split * pl.rows_cap * kPartRow : 0;
  return true;
}

// ---------------------------------------------------------------- arguments
inline int fill_seg(Seg& s, const int8_t* k, const int8_t* v, const int64_t* kvs, const void* ksc,
                    const void* vsc, const int64_t* kss, const int64_t* vss, const int* lens,
                    int cap, int nb, int units, int window, int sinks, const void* q) {
  if (cap > 0 && (!k || !v || !ksc || !vsc)) return HQ_ERR_INVALID_ARGUMENT;
  if (!kvs || !kss || !vss || cap < 0 || nb < 0 || units < 0 || window < 0 || sinks < 0)
    return HQ_ERR_INVALID_ARGUMENT;
  if (cap > 1 << 30) return HQ_ERR_UNSUPPORTED;  // key numbers and windows are ints
  if (!aligned(k, 16) || !aligned(v, 16) || kvs[0] % 16 || kvs[1] % 16 || kvs[2] % 16)
    return HQ_ERR_INVALID_ARGUMENT;
  s.k = k;
  s.v = v;
  s.sb = kvs[0];
  s.sh = kvs[1];
  s.ss = kvs[2];
  s.ksc = ksc;
  s.vsc = vsc;
  s.kscb = kss[0];
  s.ksch = kss[1];
  s.kscd = kss[2];
  s.vscb = vss[0];
  s.vsch = vss[1];
  s.vscs = vss[2];
  // An empty cache may come without scales.  The kernels read K's before they know of any key (a
  // test there took 2 % of prefix decode over 200 x 4096), so they are given readable ones; no score
  // made from them is seen.
  if (cap == 0) {
    s.ksc = q;
    s.kscb = s.ksch = s.kscd = 0;
  }
  s.lens = lens;
  s.cap = cap;
  s.nb = nb;
  s.units = units;
  // (all of a cache holds is seen at either bound, and sums of positions stay ints)
  s.window = window > 0 ? std::min(window, 1 << 30) : 1 << 30;
  s.sinks = std::min(sinks, cap);
  return HQ_OK;
}

// (an extent above 1 with a stride of 0: blocks would write the same rows)
inline bool shared_rows(int64_t n, int64_t stride) { return n > 1 && stride == 0; }

inline int check_common(const void* q, int q_dtype, const int64_t* qs, int nqs, const void* out,
                        const int64_t* os, int scale_dtype, int Hq, int Hkv, int D) {
  if (!q || !out || !qs || !os || Hq <= 0 || Hkv <= 0) return HQ_ERR_INVALID_ARGUMENT;
  if (D != kD || Hq % Hkv || Hq / Hkv > 128 || Hq > 65535 ||
      (q_dtype != HQ_DTYPE_BF16 && q_dtype != HQ_DTYPE_F16) ||
      (scale_dtype != HQ_DTYPE_F32 && scale_dtype != HQ_DTYPE_F16))
    return HQ_ERR_UNSUPPORTED;
  if (qs[nqs - 1] != 1 || os[nqs - 1] != 1 || !aligned(q, 16) || !aligned(out, 8))
    return HQ_ERR_INVALID_ARGUMENT;
  for (int i = 0; i + 1 < nqs; ++i)
    if (qs[i] % 8 || os[i] % 4) return HQ_ERR_INVALID_ARGUMENT;
  return HQ_OK;
}


inline Params make_params(const void* q, int q_dtype, int64_t qsh, int scale_dtype, int Hq, int Hkv,
                          float sm_scale, int q_quant, void* out, int64_t osb, int64_t osh,
                          int* status) {
  Params p{};
  p.q = q;
  p.qsh = qsh;
  p.q_dt = q_dtype;
  p.s_dt = scale_dtype;
  p.Hkv = Hkv;
  p.nrep = Hq / Hkv;
  p.qk_scale = sm_scale * kLog2e;
  p.q_quant = q_quant;
  p.out = out;
  p.osb = osb;
  p.osh = osh;
  p.status = status;
  return p;
}

}  // namespace rag
}  // namespace hq

using namespace hq;

extern "C" size_t hq_window_workspace_bytes(int q_dtype, int B, int Hq, int Hkv, int Sq, int S_max,
                                            int D, int window, int sinks) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq < 0 || S_max < 0 || window < 0 || sinks < 0 ||
      D != rag::kD || Hq % Hkv || Hq / Hkv > 128)
    return 0;
  if (Sq == 0) {
    rag::Stream pl;
    return rag::plan_stream(pl, q_dtype, Hkv, B, Hq / Hkv, S_max) ? std::max<size_t>(pl.bytes(), 256) : 0;
  }
  rag::Prefill pl;
  return rag::plan_prefill(pl, q_dtype, B, Hkv, Hq / Hkv, Sq, S_max, window > 0 ? window : 1 << 30, sinks)
             ? std::max<size_t>(pl.bytes(), 256)
             : 0;
}

extern "C" int hq_window_decode_int8(const void* q, int q_dtype, const int64_t q_strides[3],
                                     const int8_t* k, const int8_t* v, const int64_t kv_strides[3],
                                     const void* k_scale, const void* v_scale, int scale_dtype,
                                     const int64_t ksc_strides[3], const int64_t vsc_strides[3],
                                     const int* lens, int B, int Hq, int Hkv, int S_max, int D,
                                     int window, int sinks, float sm_scale, int q_quant, void* out,
                                     const int64_t out_strides[3], void* workspace,
                                     size_t workspace_bytes, int* status, hq_stream_t stream) {
  int rc = rag::check_common(q, q_dtype, q_strides, 3, out, out_strides, scale_dtype, Hq, Hkv, D);
  if (rc != HQ_OK) return rc;
  if (B < 0 || rag::shared_rows(B, out_strides[0]) || rag::shared_rows(Hq, out_strides[1]))
    return HQ_ERR_INVALID_ARGUMENT;
  rag::Source s{};
  s.p = rag::make_params(q, q_dtype, q_strides[1], scale_dtype, Hq, Hkv, sm_scale, q_quant, out,
                         out_strides[0], out_strides[1], status);
  rc = rag::fill_seg(s.p.seg, k, v, kv_strides, k_scale, v_scale, ksc_strides, vsc_strides, lens,
                     S_max, B, 1, window, sinks, q);
  if (rc != HQ_OK) return rc;
  if (B == 0) return HQ_OK;
  s.p.seg.qsb = q_strides[0];
  rag::Stream pl;
  if (!rag::plan_stream(pl, q_dtype, Hkv, B, Hq / Hkv, S_max)) return HQ_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < pl.bytes() || !rag::aligned(workspace, 256)) return HQ_ERR_WORKSPACE;
  rag::attach(s.p, pl, static_cast<char*>(workspace));
  s.grid = pl.grid;
  s.mt = pl.mt;
  s.per_entry = 1;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  rc = rag::run_stream(s.p, pl, st);
  return rc != HQ_OK ? rc : rag::combine<1, true>(s, s, B, 1, st);
}

extern "C" int hq_window_prefill_int8(const void* q, int q_dtype, const int64_t q_strides[4],
                                      const int8_t* k, const int8_t* v, const int64_t kv_strides[3],
                                      const void* k_scale, const void* v_scale, int scale_dtype,
                                      const int64_t ksc_strides[3], const int64_t vsc_strides[3],
                                      const int* lens, const int* q_lens, int B, int Hq, int Hkv,
                                      int Sq, int S_max, int D, int window, int sinks,
                                      float sm_scale, int q_quant, void* out,
                                      const int64_t out_strides[4], void* workspace,
                                      size_t workspace_bytes, int* status, hq_stream_t stream) {
  int rc = rag::check_common(q, q_dtype, q_strides, 4, out, out_strides, scale_dtype, Hq, Hkv, D);
  if (rc != HQ_OK) return rc;
  if (B < 0 || Sq < 0 || rag::shared_rows(B, out_strides[0]) || rag::shared_rows(Hq, out_strides[1]) ||
      rag::shared_rows(Sq, out_strides[2]))
    return HQ_ERR_INVALID_ARGUMENT;
  if (B > 65535 || int64_t(B) * Sq > 0x7fffffff) return HQ_ERR_UNSUPPORTED;
  rag::Source s{};
  s.p = rag::make_params(q, q_dtype, q_strides[1], scale_dtype, Hq, Hkv, sm_scale, q_quant, out,
                         out_strides[0], out_strides[1], status);
  rc = rag::fill_seg(s.p.seg, k, v, kv_strides, k_scale, v_scale, ksc_strides, vsc_strides, lens,
                     S_max, B, Sq, window, sinks, q);
  if (rc != HQ_OK) return rc;
  if (B == 0 || Sq == 0) return HQ_OK;
  s.p.seg.step = 1;
  s.p.seg.qsb = q_strides[0];
  s.p.seg.qsu = q_strides[2];
  s.p.osu = out_strides[2];
  s.p.q_lens = q_lens;
  rag::Prefill pl;
  if (!rag::plan_prefill(pl, q_dtype, B, Hkv, Hq / Hkv, Sq, S_max, s.p.seg.window, sinks))
    return HQ_ERR_UNSUPPORTED;
  if (pl.bytes() && (!workspace || workspace_bytes < pl.bytes() || !rag::aligned(workspace, 256)))
    return HQ_ERR_WORKSPACE;
  s.p.part = static_cast<float*>(workspace);
  s.p.rows_cap = pl.rows_cap;
  s.p.n_split = pl.n_split;
  s.p.n_rt = pl.n_rt;
  s.mt = 128 * pl.nm;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  rc = rag::tiles_prefill(s.p, pl.nm, B, st);
  if (rc != HQ_OK || pl.n_split == 1) return rc;
  return rag::combine<1, false>(s, s, B, Sq, st);
}

extern "C" size_t hq_prefix_decode_workspace_bytes(int q_dtype, int G, int B, int Hq, int Hkv,
                                                   int P_max, int S_max, int D) {
  if (G <= 0 || B <= 0 || B % G || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq / Hkv > 128 || P_max < 0 ||
      S_max < 0 || D != rag::kD)
    return 0;
  const int nrep = Hq / Hkv;
  rag::Stream a, b;
  if (!rag::plan_stream(a, q_dtype, Hkv, G, int64_t(B / G) * nrep, P_max) ||
      !rag::plan_stream(b, q_dtype, Hkv, B, nrep, S_max))
    return 0;
  return a.bytes() + b.bytes();
}

extern "C" int hq_prefix_decode_int8(
    const void* q, int q_dtype, const int64_t q_strides[3], const int8_t* pk, const int8_t* pv,
    const int64_t pkv_strides[3], const void* pk_scale, const void* pv_scale,
    const int64_t pksc_strides[3], const int64_t pvsc_strides[3], const int* prefix_lens, int G,
    int P_max, const int8_t* k, const int8_t* v, const int64_t kv_strides[3], const void* k_scale,
    const void* v_scale, const int64_t ksc_strides[3], const int64_t vsc_strides[3],
    const int* lens, int S_max, int scale_dtype, int B, int Hq, int Hkv, int D, float sm_scale,
    int q_quant, void* out, const int64_t out_strides[3], void* workspace, size_t workspace_bytes,
    int* status, hq_stream_t stream) {
  int rc = rag::check_common(q, q_dtype, q_strides, 3, out, out_strides, scale_dtype, Hq, Hkv, D);
  if (rc != HQ_OK) return rc;
  if (B < 0 || G <= 0 || B % G || rag::shared_rows(B, out_strides[0]) ||
      rag::shared_rows(Hq, out_strides[1]))
    return HQ_ERR_INVALID_ARGUMENT;
  rag::Source own{}, pre{};
  own.p = rag::make_params(q, q_dtype, q_strides[1], scale_dtype, Hq, Hkv, sm_scale, q_quant, out,
                           out_strides[0], out_strides[1], status);
  own.p.merge_all = 1;
  pre.p = own.p;
  rc = rag::fill_seg(pre.p.seg, pk, pv, pkv_strides, pk_scale, pv_scale, pksc_strides, pvsc_strides,
                     prefix_lens, P_max, G, B / G, 0, 0, q);
  if (rc == HQ_OK)
    rc = rag::fill_seg(own.p.seg, k, v, kv_strides, k_scale, v_scale, ksc_strides, vsc_strides, lens,
                       S_max, B, 1, 0, 0, q);
  if (rc != HQ_OK) return rc;
  if (B == 0) return HQ_OK;
  const int nrep = Hq / Hkv;
  rag::Stream a, b;
  if (!rag::plan_stream(a, q_dtype, Hkv, G, int64_t(B / G) * nrep, P_max) ||
      !rag::plan_stream(b, q_dtype, Hkv, B, nrep, S_max))
    return HQ_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < a.bytes() + b.bytes() || !rag::aligned(workspace, 256))
    return HQ_ERR_WORKSPACE;
  rag::attach(pre.p, a, static_cast<char*>(workspace));
  rag::attach(own.p, b, static_cast<char*>(workspace) + a.bytes());
  pre.p.seg.qsb = q_strides[0] * (B / G);
  pre.p.seg.qsu = q_strides[0];
  own.p.seg.qsb = q_strides[0];
  pre.grid = a.grid;
  pre.mt = a.mt;
  pre.per_entry = B / G;
  own.grid = b.grid;
  own.mt = b.mt;
  own.per_entry = 1;
  own.p.after = 1;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  rc = rag::run_stream(pre.p, a, st);
  if (rc == HQ_OK) rc = rag::run_stream(own.p, b, st);
  return rc != HQ_OK ? rc : rag::combine<2, true>(own, pre, B, 1, st);
}
