// What the ragged-batch attention kernels share: the description of a call, the pieces of work
// its blocks walk, the partial states and output rows.  Used by ragged_attn.cu (tcgen05 kernel),
// ragged_rows.cu (decode with few rows per kv head) and ragged_api.cu (plans, joining of partial
// states, entry points).
#pragma once

#include <atomic>

#include "hq_common.cuh"

namespace hq {
int current_sm_count();

namespace rag {

constexpr int kD = 128;
constexpr int kBN = 128;                  // keys per tile
constexpr int kMaxEntries = 1024;         // sequences (or groups) of one call
constexpr int kPartRow = kD + 4;          // partial rows: m, l, two pad words, o
constexpr float kLog2e = 1.4426950408889634f;

// One set of keys and the rows that read it.
struct Seg {
  const int8_t* k;
  const int8_t* v;
  int64_t sb, sh, ss;                     // strides of both (b, h, token)
  const void* ksc;
  const void* vsc;
  int64_t kscb, ksch, kscd, vscb, vsch, vscs;
  const int* lens;                        // tokens held, per entry; null: cap
  int cap;
  int nb;                                 // entries (sequences, or groups)
  int units;                              // queries per entry
  int step;                               // 1: query u stands u positions after query 0
  int64_t qsb, qsu;
  int window, sinks;
};

struct Params {
  Seg seg;
  const void* q;
  int64_t qsh;
  int q_dt, s_dt;
  int Hkv, nrep;
  float qk_scale;                         // sm_scale * log2(e)
  int q_quant;
  const int* q_lens;                      // prefill: queries per sequence; null: all
  void* out;                              // rows [b][u][h]
  int64_t osb, osu, osh;
  float* part;                            // partial states
  int* cum;                               // STREAM: first tile of each entry, for combine_kernel
  int* status;
  int n_split, n_rt;                      // prefill grid: splits, row tiles
  int merge_all;                          // every piece goes through combine_kernel
  int rows_cap;                           // partial rows per piece
  int min_tiles;                          // STREAM: least tiles per block
  int after;                              // launched beside the kernel before: ends after it
};

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// ---------------------------------------------------------------- pieces of work
// The keys of one row tile, numbered v = 0 .. nv - 1: the sinks 0 .. ns - 1, then numbers up to
// nsp that nobody sees (where the copies want the next run to start at a multiple of 8), then
// key v + sh.
struct Keys {
  int pos0;        // position of the entry's query 0
  int ns, nsp, sh, nv, nt;
  __device__ __forceinline__ int key(int v) const { return v < nsp ? v : v + sh; }
  __device__ __forceinline__ bool padding(int v) const { return v >= ns && v < nsp; }
};
__device__ __forceinline__ int seg_len(const Seg& s, int b) {
  return s.lens ? min(max(s.lens[b], 0), s.cap) : s.cap;
}
// n tokens held, nq queries of which rows u_lo .. u_hi are in the tile
template <int AL>
__device__ __forceinline__ Keys make_keys(const Seg& s, int n, int nq, int u_lo, int u_hi) {
  Keys k;
  k.pos0 = s.step ? n - nq : n - 1;
  const int p_lo = k.pos0 + (s.step ? u_lo : 0), p_hi = k.pos0 + (s.step ? u_hi : 0);
  const int w0 = max(0, p_lo - s.window + 1), nsp = (s.sinks + AL - 1) / AL * AL;
  // apart: two runs; else one run of keys (of which sinks .. w0 - 1 may be unseen)
  const bool apart = w0 > nsp, gap = w0 > s.sinks;
  k.ns = gap ? s.sinks : 0;
  k.nsp = apart ? nsp : gap ? w0 : 0;
  k.sh = apart ? w0 - nsp : 0;
  k.nv = max(p_hi + 1 - k.sh, 0);
  k.nt = (k.nv + kBN - 1) / kBN;
  return k;
}
struct Piece {
  int b, kvh, row0, rows;
  Keys key;
  int t0, t1;
  int slot;        // -1: final output
};
__device__ __host__ __forceinline__ int row_tiles(int rows, int mt) { return (rows + mt - 1) / mt; }

// STREAM: keys of entry e; tiles of one row tile (0: the call is answered by combine_kernel)
template <int AL>
__device__ __forceinline__ Keys entry_keys(const Params& p, int e) {
  Keys k = make_keys<AL>(p.seg, seg_len(p.seg, e), p.seg.units, 0, 0);
  if (!p.merge_all) k.nt = max(k.nt, 1);
  return k;
}
// cum[e]: first tile of entry e in the line of all tiles (shared memory, nb + 1 words; ends
// with a block barrier).  Block 0 leaves a copy for combine_kernel.
template <int MT, int AL>
__device__ __forceinline__ void build_cum(const Params& p, int* cum, int n_threads) {
  const int ne = p.seg.nb, per = p.Hkv * row_tiles(p.seg.units * p.nrep, MT);
  if (ne <= 32) {  // one warp does it alone
    if (threadIdx.x < 32) {
      int x = threadIdx.x < ne ? entry_keys<AL>(p, threadIdx.x).nt * per : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (threadIdx.x >= o) x += y;
      }
      if (threadIdx.x == 0) cum[0] = 0;
      if (threadIdx.x < ne) cum[threadIdx.x + 1] = x;
    }
  } else {
    for (int e = threadIdx.x; e < ne; e += n_threads) cum[e + 1] = entry_keys<AL>(p, e).nt * per;
    __syncthreads();
    if (threadIdx.x < 32) {
      const int lane = threadIdx.x;
      int run = 0;
      if (lane == 0) cum[0] = 0;
#pragma unroll 1
      for (int e0 = 0; e0 < ne; e0 += 32) {
        int x = e0 + lane < ne ? cum[e0 + lane + 1] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        if (e0 + lane < ne) cum[e0 + lane + 1] = run + x;
        run += __shfl_sync(0xffffffffu, x, 31);
      }
    }
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= ne; e += n_threads) p.cum[e] = cum[e];
}
__device__ __forceinline__ int tiles_per_block(const Params& p, int total, int grid) {
  return max(p.min_tiles, (total + grid - 1) / grid);
}

// The pieces of one block, in order.  STREAM: an equal run of the line of tiles, cut where the
// units (entry, row tile, kv head) end; the state is the unit at hand, stepped from one to the
// next (a divide and two modulos per piece cost 2400 cycles of a cold call).
struct Walk {
  int cur, end;                  // tiles of the line
  int e, rt, kvh, first;         // the unit, its first tile
  Keys key;
};
template <int MT, bool STREAM, int AL>
__device__ __forceinline__ Walk walk_start(const Params& p, const int* cum) {
  Walk k{};
  if constexpr (STREAM) {
    const int ne = p.seg.nb, total = cum[ne];
    const int per = tiles_per_block(p, total, static_cast<int>(gridDim.x));
    k.cur = static_cast<int>(min(static_cast<int64_t>(blockIdx.x) * per, static_cast<int64_t>(total)));
    k.end = static_cast<int>(min(static_cast<int64_t>(k.cur) + per, static_cast<int64_t>(total)));
    if (k.cur >= k.end) return k;
    // the entry that holds tile cur: cum[e] <= cur < cum[e + 1]
    int lo = 0, hi = ne - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cum[mid] <= k.cur) lo = mid; else hi = mid - 1;
    }
    k.e = lo;
    k.key = entry_keys<AL>(p, lo);
    const uint32_t idx = static_cast<uint32_t>(k.cur - cum[lo]) / static_cast<uint32_t>(k.key.nt);
    k.rt = idx / static_cast<uint32_t>(p.Hkv);
    k.kvh = idx - k.rt * p.Hkv;
    k.first = cum[lo] + idx * k.key.nt;
  } else {
    k.end = 1;
  }
  return k;
}
template <int MT, bool STREAM, int AL>
__device__ __forceinline__ bool walk_next(Walk& k, const Params& p, const int* cum, Piece& w) {
  if (k.cur >= k.end) return false;
  const Seg& s = p.seg;
  if constexpr (STREAM) {
    const int rows = s.units * p.nrep, n_rt = MT == 128 && rows <= 128 ? 1 : row_tiles(rows, MT);
    w.b = k.e;
    w.kvh = k.kvh;
    w.row0 = k.rt * MT;
    w.rows = min(MT, rows - w.row0);
    w.key = k.key;
    w.t0 = k.cur - k.first;
    w.t1 = min(k.key.nt, w.t0 + k.end - k.cur);
    w.slot = !p.merge_all && w.t0 == 0 && w.t1 == k.key.nt
                 ? -1
                 : (k.e * n_rt + k.rt) * p.Hkv + k.kvh + static_cast<int>(blockIdx.x);
    k.cur = k.first + w.t1;
    if (w.t1 == k.key.nt && k.cur < k.end) {  // on to the next unit
      k.first = k.cur;
      if (++k.kvh == p.Hkv) {
        k.kvh = 0;
        if (++k.rt == n_rt) {
          k.rt = 0;
          do ++k.e; while (cum[k.e + 1] == k.cur);
          k.key = entry_keys<AL>(p, k.e);
        }
      }
    }
  } else {
    k.cur = 1;
    // longest row tiles (the last ones of a causal chunk) first
    const int rq = static_cast<uint32_t>(blockIdx.y) / static_cast<uint32_t>(p.Hkv);
    const int rt = p.n_rt - 1 - rq;
    const int b = blockIdx.z;
    const int nq = p.q_lens ? min(max(p.q_lens[b], 0), s.units) : s.units;
    w.b = b;
    w.kvh = static_cast<int>(blockIdx.y) - rq * p.Hkv;
    w.row0 = rt * MT;
    w.rows = min(MT, nq * p.nrep - w.row0);
    if (w.rows <= 0) return false;
    w.key = make_keys<AL>(s, seg_len(s, b), nq, static_cast<uint32_t>(w.row0) / static_cast<uint32_t>(p.nrep),
                          static_cast<uint32_t>(w.row0 + w.rows - 1) / static_cast<uint32_t>(p.nrep));
    const uint32_t nt = max(w.key.nt, 1), ns = p.n_split, split = blockIdx.x;  // nt < 2^24, ns <= 16
    w.t0 = static_cast<int>(nt * split / ns);
    w.t1 = static_cast<int>(nt * (split + 1) / ns);
    w.slot = ns == 1 ? -1 : ((b * p.Hkv + w.kvh) * p.n_rt + rt) * static_cast<int>(ns) + static_cast<int>(split);
  }
  return true;
}

__device__ __forceinline__ float* part_row(const Params& p, int slot, int r) {
  return p.part + (static_cast<int64_t>(slot) * p.rows_cap + r) * kPartRow;
}

// Stores 4 consecutive values of an output row.
__device__ __forceinline__ void store4(void* row, int dt, int d, float a, float b, float c, float e) {
  uint2 w;
  if (dt == HQ_DTYPE_BF16) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, e);
    w = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  } else {
    w = make_uint2(pack_h2(a, b), pack_h2(c, e));
  }
  *reinterpret_cast<uint2*>(static_cast<char*>(row) + 2 * d) = w;
}
__device__ __forceinline__ uint32_t pack_pair(float a, float b, int dt) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
  return dt == HQ_DTYPE_BF16 ? *reinterpret_cast<const uint32_t*>(&x) : pack_h2(a, b);
}
__device__ __forceinline__ char* out_row(const Params& p, int b, int u, int h) {
  return static_cast<char*>(p.out) + 2 * (b * p.osb + u * p.osu + h * p.osh);
}

// A scale's bits, and its value.  Apart, because a conversion behind the load's own branch would
// wait there for the memory: 1300 cycles a tile where the loads run two tiles ahead.
__device__ __forceinline__ uint32_t load_bits(const void* p, int64_t i, int dt) {
  return dt == HQ_DTYPE_F32 ? static_cast<const uint32_t*>(p)[i]
                            : static_cast<uint32_t>(static_cast<const unsigned short*>(p)[i]);
}
__device__ __forceinline__ float scale_of(uint32_t bits, int dt) {
  return dt == HQ_DTYPE_F32 ? __uint_as_float(bits)
                            : __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

// Sets a kernel's dynamic shared-memory limit once per device.
template <typename K>
int set_smem(K kern, int bytes, std::atomic<uint64_t>& ready) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = (dev >= 0 && dev < 64) ? (uint64_t(1) << dev) : 0;
  if (!bit || !(ready.load(std::memory_order_acquire) & bit)) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    ready.fetch_or(bit, std::memory_order_acq_rel);
  }
  return HQ_OK;
}

// Launches a kernel of Params (and more); with p.after it may start beside the kernel before it on the
// stream (which it does not read from), and completes after it.
template <typename K, typename... A>
int launch_after(K kern, dim3 grid, int threads, int smem, cudaStream_t st, const Params& p, const A&... more) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.after ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, more...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return static_cast<int>(e);
  }
  return HQ_OK;
}

// Launches of the kernels (ragged_attn.cu, ragged_rows.cu).
int tiles_stream(const Params& p, int nm, int grid, cudaStream_t st);
int tiles_prefill(const Params& p, int nm, int B, cudaStream_t st);
int rows_stream(const Params& p, int grid, cudaStream_t st);
constexpr int kMaxRows = 4;  // rows per kv head that ragged_rows.cu takes

}  // namespace rag
}  // namespace hq
