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
// float64 quotient: one rounding of the exact value.
#include <algorithm>

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
