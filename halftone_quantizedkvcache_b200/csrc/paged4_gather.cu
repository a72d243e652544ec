// Tokens of a paged 4-bit cache as packed 16-bit rows (sm_100a): row cu[b] + i takes token
// first[b] + i of sequence b, the value s * code rounded once to the row's type.
//
// Bound by memory: 144 bytes read and 512 written per token and kv head (8 x 8192 tokens of 8 heads, bf16:
// 64 us, 5.3 TB/s, 0.82 of a copy's rate).  16 lanes hold a row (a word of 8 codes each); a half-warp takes one
// row and all of its heads, K and V.
#include <algorithm>

#include "paged4.cuh"

namespace hq {
int current_sm_count();

namespace p4 {

struct GatherParams {
  Pages pg;
  int T, B, Hkv;
  const int* cu;
  const int* lens;
  const int* first;                       // null: 0
  void* k_out;
  void* v_out;
  int64_t ks[2], vs[2];
  int zero_rest;                          // rows that no token goes to become zeros
  int* status;
  int heads_per_block, groups;
};

// The values of a word of 8 codes: codes i and i + 4 under the exponent of 1024 are float16 numbers; float16
// values are their products with the scale, bf16 those of float32 (both exact before the one rounding).
template <int DT>
__device__ __forceinline__ uint4 values8(uint32_t w, __half s) {
  const __half2 off = __float2half2_rn(1032.0f);
  __half2 c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u;
    c[i] = __hsub2(*reinterpret_cast<const __half2*>(&x), off);
  }
  if constexpr (DT == HQ_DTYPE_F16) {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 x = __hmul2(c[i], __half2half2(s));
      v[i] = *reinterpret_cast<const uint32_t*>(&x);
    }
    return make_uint4(prmt(v[0], v[1], 0x5410u), prmt(v[2], v[3], 0x5410u), prmt(v[0], v[1], 0x7632u), prmt(v[2], v[3], 0x7632u));
  } else {
    const float sf = __half2float(s);
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 a = __half22float2(c[2 * i]), b = __half22float2(c[2 * i + 1]);
      const __nv_bfloat162 lo = __floats2bfloat162_rn(a.x * sf, b.x * sf), hi = __floats2bfloat162_rn(a.y * sf, b.y * sf);
      out[i] = *reinterpret_cast<const uint32_t*>(&lo);
      out[i + 2] = *reinterpret_cast<const uint32_t*>(&hi);
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
  }
}

constexpr int kGThreads = 256;
constexpr int kGRows = kGThreads / 16;

template <int DT>
__global__ void __launch_bounds__(kGThreads) gather_kernel(const __grid_constant__ GatherParams p) {
  const int tid = threadIdx.x, lane = tid & 31, sub = tid >> 4, l = lane & 15;
  const int group = static_cast<int>(blockIdx.x % p.groups);
  const int64_t row64 = static_cast<int64_t>(blockIdx.x / p.groups) * kGRows + sub;
  const bool here = row64 < p.T;
  const int row = static_cast<int>(here ? row64 : p.T - 1);
  const int b = find_seq(p.cu, p.B, row);
  bool held = here && b < p.B;
  int pid = 0;
  int64_t at = 0;
  if (held) {
    const int64_t cap = static_cast<int64_t>(p.pg.max_pages) << p.pg.page_log;
    const int64_t i = row - static_cast<int64_t>(p.cu[b]);
    at = i + (p.first ? max(p.first[b], 0) : 0);
    held = i >= 0 && at < min(static_cast<int64_t>(max(p.lens[b], 0)), cap);
    if (held) {
      pid = p.pg.tables[b * p.pg.tstride + (at >> p.pg.page_log)];
      if (pid < 0 || pid >= p.pg.n_pages) {
        if (l == 0) report_error(p.status, HQ_ERR_INVALID_ARGUMENT);
        held = false;
      }
    }
  }
  if (!held && !(here && p.zero_rest)) return;
  const int place = static_cast<int>(at) & (p.pg.page - 1);
  const int h0 = group * p.heads_per_block, h1 = min(p.Hkv, h0 + p.heads_per_block);
  const int64_t cat = pid * p.pg.cp + place * kRowB + word_at(place, l >> 2, l & 3);
  const int64_t sat = pid * p.pg.sp + place * 4 + (l >> 2);
#pragma unroll 1  // (two heads at once: fewer warps fit, 8 x 8192 tokens 64 to 70 us)
  for (int h = h0; h < h1; ++h) {
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if (held) {
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(p.pg.k + cat + h * p.pg.ch);
      const uint32_t vw = *reinterpret_cast<const uint32_t*>(p.pg.v + cat + h * p.pg.ch);
      const __half ks = p.pg.ksc[sat + h * p.pg.sh], vs = p.pg.vsc[sat + h * p.pg.sh];
      k = values8<DT>(kw, ks);
      v = values8<DT>(vw, vs);
    }
    *reinterpret_cast<uint4*>(static_cast<char*>(p.k_out) + 2 * (row * p.ks[0] + h * p.ks[1] + 8 * l)) = k;
    *reinterpret_cast<uint4*>(static_cast<char*>(p.v_out) + 2 * (row * p.vs[0] + h * p.vs[1] + 8 * l)) = v;
  }
}

}  // namespace p4
}  // namespace hq

using namespace hq;

extern "C" int hq_paged4_gather(const hq_paged4_gather_args* args) {
  if (!args) return HQ_ERR_INVALID_ARGUMENT;
  const hq_paged4_gather_args& a = *args;
  if (a.T < 0 || a.B < 0 || a.Hkv <= 0 || !a.cu_seqlens) return HQ_ERR_INVALID_ARGUMENT;
  if (a.D != p4::kD || (a.out_dtype != HQ_DTYPE_BF16 && a.out_dtype != HQ_DTYPE_F16) || a.Hkv > 65535) return HQ_ERR_UNSUPPORTED;
  const int rc = p4::check_pages(a.k_codes, a.v_codes, a.k_scale, a.v_scale, a.code_strides, a.scale_strides, a.n_pages,
                                 a.page_size, a.tables, a.table_stride, a.max_pages, a.B, a.Hkv);
  if (rc != HQ_OK) return rc;
  if (a.T == 0) return HQ_OK;
  auto al = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
  if (!a.k_out || !a.v_out || (a.B > 0 && !a.lens) || !al(a.k_out) || !al(a.v_out) ||
      a.k_strides[0] % 8 || a.k_strides[1] % 8 || a.v_strides[0] % 8 || a.v_strides[1] % 8)
    return HQ_ERR_INVALID_ARGUMENT;
  const Rows ko = packed_rows(a.k_out, a.T, a.Hkv, a.k_strides), vo = packed_rows(a.v_out, a.T, a.Hkv, a.v_strides);
  if (rows_meet(ko) || rows_meet(vo) || rows_meet(ko, vo)) return HQ_ERR_INVALID_ARGUMENT;
  p4::GatherParams p{};
  p.pg = p4::make_pages(a.k_codes, a.v_codes, a.k_scale, a.v_scale, a.code_strides, a.scale_strides, a.n_pages, a.page_size,
                        a.tables, a.table_stride, a.max_pages);
  p.T = a.T;
  p.B = a.B;
  p.Hkv = a.Hkv;
  p.cu = a.cu_seqlens;
  p.lens = a.lens;
  p.first = a.first;
  p.k_out = a.k_out;
  p.v_out = a.v_out;
  for (int i = 0; i < 2; ++i) {
    p.ks[i] = a.k_strides[i];
    p.vs[i] = a.v_strides[i];
  }
  p.zero_rest = a.zero_rest;
  p.status = a.status;
  const int64_t blocks = (static_cast<int64_t>(a.T) + p4::kGRows - 1) / p4::kGRows;
  // a row's heads stay together as long as that leaves 4 blocks an SM
  const int64_t want = std::max<int64_t>(1, 4LL * current_sm_count() / blocks);
  const int groups = static_cast<int>(std::min<int64_t>(a.Hkv, want));
  p.heads_per_block = (a.Hkv + groups - 1) / groups;
  p.groups = (a.Hkv + p.heads_per_block - 1) / p.heads_per_block;
  if (blocks * p.groups > 0x7fffffff) return HQ_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(a.stream);
  const unsigned grid = static_cast<unsigned>(blocks * p.groups);
  if (a.out_dtype == HQ_DTYPE_BF16) p4::gather_kernel<HQ_DTYPE_BF16><<<grid, p4::kGThreads, 0, st>>>(p);
  else p4::gather_kernel<HQ_DTYPE_F16><<<grid, p4::kGThreads, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? HQ_OK : static_cast<int>(e);
}
