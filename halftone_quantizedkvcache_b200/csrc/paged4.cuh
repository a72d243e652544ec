// The paged cache held in 4 bits: its layout, and what its kernels share (paged4_append.cu,
// paged4_decode.cu, paged4_gather.cu).
//
// Per token and kv head 128 channels in 4 groups of 32: scale s = f16(amax / 7.5), at most 65504 (and NaN for
// a group that holds an infinity or NaN), codes clamp(rint(x / s), -8, 7), values s * code.  7.5 puts both ends of a group half a step from a code,
// so that no value is off by more than half a step (amax / 8 or amax / 7 would clip one end or leave a
// code unused).  A page holds `page` tokens of every kv head: codes [page][64 bytes] and scales
// [page][4] of one head are each one piece of memory, which a bulk copy takes whole.
//
// A row's 64 bytes: the 16 bytes at position p hold chunk j = p ^ 2 ((t >> 1) & 1), t the token's
// place in its page; the chunk's word g has channels 32 g + 8 j + i, i = 0 .. 7, as code + 8 in bits
// 4 i .. 4 i + 3.  A lane of the decode kernel so finds one eighth-row of every group in one 16-byte
// load, and the swizzle keeps the loads of 8 lanes in different banks for K (two tokens, all chunks)
// and for V (four tokens, two chunks).
#pragma once

#include <cmath>

#include "hq_common.cuh"
#include "rows.cuh"

namespace hq {
namespace p4 {

constexpr int kD = 128;
constexpr int kRowB = 64;                 // bytes of a token's codes
constexpr int kScaleB = 8;                // bytes of a token's scales

struct Pages {
  uint8_t* k;
  uint8_t* v;
  __half* ksc;
  __half* vsc;
  int64_t cp, ch;                         // codes: strides of page and head, in bytes
  int64_t sp, sh;                         // scales: in elements
  int n_pages;
  int page, page_log;                     // tokens a page, a power of two
  const int* tables;                      // [B][max_pages]
  int64_t tstride;
  int max_pages;
};

// Byte position of word (g, j) in a code row at place t of its page.
__device__ __forceinline__ int word_at(int t, int g, int j) { return 16 * (j ^ (t & 2)) + 4 * g; }

// Which of the sequences of cu[0 .. B] holds each of the warp's rows `at`: the number of starts
// cu[1 .. B] at or below it (B: behind the last).  All lanes together; rows differ from half-warp to
// half-warp at most.  Linear in B: 8192 one-token sequences are appended in 72 us, in 44 without starts.
__device__ __forceinline__ int find_seq(const int* cu, int B, int at) {
  const int lane = threadIdx.x & 31;
  const int lo = __shfl_sync(0xffffffffu, at, 0), hi = __shfl_sync(0xffffffffu, at, 16);
  int n_lo = 0, n_hi = 0;
  for (int i = lane; i - lane < B; i += 32) {
    const int c = i < B ? cu[i + 1] : 0x7fffffff;
    n_lo += __popc(__ballot_sync(0xffffffffu, c <= lo));
    n_hi += __popc(__ballot_sync(0xffffffffu, c <= hi));
  }
  return lane < 16 ? n_lo : n_hi;
}

// Host side: checks of a cache's arguments.
inline int check_pages(const void* k, const void* v, const void* ks, const void* vs, const int64_t cs[2],
                       const int64_t ss[2], int n_pages, int page, const int* tables, int64_t tstride,
                       int max_pages, int B, int Hkv) {
  if (!cs || !ss || n_pages < 0 || max_pages < 0 || B < 0 || Hkv <= 0 || tstride < 0) return HQ_ERR_INVALID_ARGUMENT;
  if (page < 16 || page > 256 || (page & (page - 1))) return HQ_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(max_pages) * page > (1 << 30)) return HQ_ERR_UNSUPPORTED;
  if (B > 0 && max_pages > 0 && !tables) return HQ_ERR_INVALID_ARGUMENT;
  if (n_pages > 0) {
    if (!k || !v || !ks || !vs) return HQ_ERR_INVALID_ARGUMENT;
    auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    if (!al(k) || !al(v) || !al(ks) || !al(vs) || cs[0] % 16 || cs[1] % 16 || ss[0] % 8 || ss[1] % 8)
      return HQ_ERR_INVALID_ARGUMENT;
    if (cs[0] >> 31 || ss[0] >> 30) return HQ_ERR_UNSUPPORTED;  // page strides below 2 GB
    // pages and heads have memory of their own
    if ((n_pages > 1 && cs[0] < static_cast<int64_t>(page) * kRowB) || (Hkv > 1 && cs[1] < static_cast<int64_t>(page) * kRowB) ||
        (n_pages > 1 && ss[0] < static_cast<int64_t>(page) * 4) || (Hkv > 1 && ss[1] < static_cast<int64_t>(page) * 4))
      return HQ_ERR_INVALID_ARGUMENT;
  }
  return HQ_OK;
}
// Pages and heads of K and V (codes or scales: a row of `row` bytes per token, strides in units of `unit`
// bytes) that share no memory.
inline bool own_memory(const void* k, const void* v, const int64_t st[2], int unit, int row, int n_pages, int Hkv, int page) {
  const Rows a = rows_of(k, n_pages, Hkv, unit * st[0], unit * st[1], int64_t(row) * page);
  Rows b = a;
  b.base = v;
  return !rows_meet(a) && !rows_meet(a, b);
}
inline Pages make_pages(const void* k, const void* v, const void* ks, const void* vs, const int64_t cs[2],
                        const int64_t ss[2], int n_pages, int page, const int* tables, int64_t tstride,
                        int max_pages) {
  Pages p{};
  p.k = static_cast<uint8_t*>(const_cast<void*>(k));
  p.v = static_cast<uint8_t*>(const_cast<void*>(v));
  p.ksc = static_cast<__half*>(const_cast<void*>(ks));
  p.vsc = static_cast<__half*>(const_cast<void*>(vs));
  p.cp = cs[0];
  p.ch = cs[1];
  p.sp = ss[0];
  p.sh = ss[1];
  p.n_pages = n_pages;
  p.page = page;
  p.page_log = 31 - __builtin_clz(page);
  p.tables = tables;
  p.tstride = tstride;
  p.max_pages = max_pages;
  return p;
}

}  // namespace p4
}  // namespace hq
