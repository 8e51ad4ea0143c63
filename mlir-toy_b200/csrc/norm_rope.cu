// Norm and position rotation of queries and keys, and their append to the paged KV cache.
//
// For a row x of one token and head, with weights w (or none: y = x), frequencies f and the token's position p:
//
//   y = x * rsqrt(mean(x^2) + eps) * w          over the D elements of the row
//   (y1, y2) <- (y1 cos a - y2 sin a, y2 cos a + y1 sin a),  a = p * f[i],  i < rot / 2
//
// where the pair is (i, i + rot/2) or (2i, 2i+1); elements from rot on pass through.  Everything is fp32 and rounded
// once, on the way out.  The angle is reduced to a fraction of a turn in fp64: p * f in fp32 would be off by 0.06 rad at
// position 10^6.
//
// One CTA per token (and, for few tokens, per group of its rows): a row is read by G lanes, 8 elements each, so a thread
// holds U rows at once and its loads are in flight while 64 threads compute the token's sines and cosines.  A pair's
// other half is eight shuffles away; a row is read and written once, so the call is bound by HBM.
#include "nb200_common.cuh"

namespace nb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;          // rot <= 256
constexpr int kPageRows = 64;
constexpr int kCacheD = 128;

enum : int { kErrTable = 22, kErrSlot = 23 };   // see nb200_status_read

struct Strides {
  long long b, t, h;                   // batch, token, head, in elements
};
struct Args {
  const void *q, *k, *v;               // v: append only
  void *q_out, *k_out;                 // k_out: without append
  Strides sq, sk, sv, sqo, sko;
  const void *wq, *wk;                 // [D] or null
  const float *inv_freq;               // [rot / 2]
  const int *positions;                // without append
  long long positions_b;
  int S, Hq, Hkv, D, rot, interleaved;
  float eps, inv_d;
  // append
  void *k_pages, *v_pages;
  const int *block_table, *cu_seqlens, *seq_lens;
  int B, num_pages, max_pages;
  int *status;
};

// Eight consecutive elements of a row as they are stored.
template <int DT> struct Raw {
  uint4 w[DT == NB200_F32 ? 2 : 1];
};
template <int DT> __device__ __forceinline__ Raw<DT> load_raw(const void *base, long long elem) {
  Raw<DT> r;
  const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const char *>(base) + elem * (DT == NB200_F32 ? 4 : 2));
#pragma unroll
  for (int i = 0; i < (DT == NB200_F32 ? 2 : 1); ++i) r.w[i] = p[i];
  return r;
}
template <int DT> __device__ __forceinline__ void store_raw(void *base, long long elem, const Raw<DT> &r) {
  uint4 *p = reinterpret_cast<uint4 *>(static_cast<char *>(base) + elem * (DT == NB200_F32 ? 4 : 2));
#pragma unroll
  for (int i = 0; i < (DT == NB200_F32 ? 2 : 1); ++i) p[i] = r.w[i];
}
template <int DT> __device__ __forceinline__ void to_float(const Raw<DT> &r, float (&y)[8]) {
  const uint32_t *w = reinterpret_cast<const uint32_t *>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == NB200_F32) {
      y[2 * i] = __uint_as_float(w[2 * i]);
      y[2 * i + 1] = __uint_as_float(w[2 * i + 1]);
    } else {
      const float2 f = unpack2<DT>(w[i]);
      y[2 * i] = f.x;
      y[2 * i + 1] = f.y;
    }
  }
}
template <int DT> __device__ __forceinline__ Raw<DT> from_float(const float (&y)[8]) {
  Raw<DT> r;
  uint32_t *w = reinterpret_cast<uint32_t *>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == NB200_F32) {
      w[2 * i] = __float_as_uint(y[2 * i]);
      w[2 * i + 1] = __float_as_uint(y[2 * i + 1]);
    } else {
      w[i] = pack2<DT>(y[2 * i], y[2 * i + 1]);
    }
  }
  return r;
}

__device__ __forceinline__ void report(int *status, int code, int detail, int detail2) {
  if (status && atomicCAS(status, 0, code) == 0) {
    status[1] = static_cast<int>(blockIdx.x);
    status[2] = detail;
    status[3] = detail2;
  }
}

// Rows of a token: Hq queries, then Hkv keys, then (append) Hkv values.
template <int DT, int G, int U, bool APPEND>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const Args a) {
  constexpr int kRows = kThreads / G;
  __shared__ float2 turn[kMaxHalf];                       // (cos, sin) of the token's angles
  const long long t = blockIdx.x;
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  const int row0 = blockIdx.y * (kRows * U) + sub;
  const int rows = a.Hq + (APPEND ? 2 : 1) * a.Hkv;
  const int c0 = lane * 8;
  const bool in_row = c0 < a.D;
  const long long bt = APPEND ? 0 : t / a.S, st = APPEND ? t : t % a.S;

  Raw<DT> raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int row = row0 + u * kRows;
    raw[u] = Raw<DT>{};
    if (in_row && row < rows) {
      if (row < a.Hq)
        raw[u] = load_raw<DT>(a.q, bt * a.sq.b + st * a.sq.t + row * a.sq.h + c0);
      else if (!APPEND || row < a.Hq + a.Hkv)
        raw[u] = load_raw<DT>(a.k, bt * a.sk.b + st * a.sk.t + (row - a.Hq) * a.sk.h + c0);
      else
        raw[u] = load_raw<DT>(a.v, st * a.sv.t + (row - a.Hq - a.Hkv) * a.sv.h + c0);
    }
  }

  int pos = 0;
  long long slot_base = 0;                                // element offset of (page, head 0, row) in the pools
  if constexpr (APPEND) {
    // the sequence whose tokens include t: one past the last entry of cu_seqlens that is <= t
    int below = 0;
    for (int i = 0; i <= a.B; i += kThreads)
      below += __syncthreads_count(i + static_cast<int>(threadIdx.x) <= a.B && a.cu_seqlens[min(i + static_cast<int>(threadIdx.x), a.B)] <= t);
    const int b = below - 1;
    if (b < 0 || b >= a.B) return;                        // a row behind the last sequence: left as it was
    const int first = a.cu_seqlens[b], end = a.cu_seqlens[b + 1];
    if (t < first || t >= end) return;                    // cu_seqlens is not a running sum
    const long long p = static_cast<long long>(a.seq_lens[b]) - end + t;
    if (p < 0 || p >= static_cast<long long>(a.max_pages) * kPageRows) {
      if (threadIdx.x == 0 && blockIdx.y == 0) report(a.status, kErrSlot, static_cast<int>(t), static_cast<int>(p));
      return;
    }
    pos = static_cast<int>(p);
    const int page = a.block_table[static_cast<long long>(b) * a.max_pages + pos / kPageRows];
    if (page < 0 || page >= a.num_pages) {
      if (threadIdx.x == 0 && blockIdx.y == 0) report(a.status, kErrTable, page, static_cast<int>(threadIdx.x));
      return;
    }
    slot_base = (static_cast<long long>(page) * a.Hkv * kPageRows + pos % kPageRows) * kCacheD;
  } else {
    pos = a.positions[bt * a.positions_b + st];
  }

  for (int i = threadIdx.x; i < a.rot / 2; i += kThreads) {
    const double turns = static_cast<double>(pos) * static_cast<double>(a.inv_freq[i]) * 0.15915494309189535;   // 1 / 2 pi
    float s, c;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
    turn[i] = make_float2(c, s);
  }
  __syncthreads();

#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int row = row0 + u * kRows;
    const bool is_q = row < a.Hq, is_v = APPEND && row >= a.Hq + a.Hkv;
    const void *w = is_q ? a.wq : a.wk;
    float y[8];
    to_float<DT>(raw[u], y);
    if (a.wq || a.wk) {                                   // uniform: every lane takes part in the sum
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(y[i], y[i], ss);
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (w && in_row) {
        const float r = rsqrtf(fmaf(ss, a.inv_d, a.eps));
        float g[8];
        to_float<DT>(load_raw<DT>(w, c0), g);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * r * g[i];
      }
    }
    if (a.interleaved) {
      if (c0 < a.rot) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 cs = turn[c0 / 2 + i];
          const float y1 = y[2 * i], y2 = y[2 * i + 1];
          y[2 * i] = y1 * cs.x - y2 * cs.y;
          y[2 * i + 1] = y2 * cs.x + y1 * cs.y;
        }
      }
    } else {
      // the other half of the pairs of this lane's 8 elements sits rot / 16 lanes up or down
      const int half = a.rot / 16;
      const bool low = lane < half;
      const int other = low ? lane + half : (lane < 2 * half ? lane - half : lane);
      float z[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = __shfl_sync(0xffffffffu, y[i], other, G);
      if (lane < 2 * half) {
        const int i0 = (low ? lane : lane - half) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 cs = turn[i0 + i];
          y[i] = fmaf(low ? -z[i] : z[i], cs.y, y[i] * cs.x);
        }
      }
    }
    if (in_row && row < rows) {
      if (is_q)
        store_raw<DT>(a.q_out, bt * a.sqo.b + st * a.sqo.t + row * a.sqo.h + c0, from_float<DT>(y));
      else if constexpr (!APPEND)
        store_raw<DT>(a.k_out, bt * a.sko.b + st * a.sko.t + (row - a.Hq) * a.sko.h + c0, from_float<DT>(y));
      else if (is_v)
        store_raw<DT>(a.v_pages, slot_base + static_cast<long long>(row - a.Hq - a.Hkv) * (kPageRows * kCacheD) + c0, raw[u]);
      else
        store_raw<DT>(a.k_pages, slot_base + static_cast<long long>(row - a.Hq) * (kPageRows * kCacheD) + c0, from_float<DT>(y));
    }
  }
}

template <int DT, int G, int U, bool APPEND> int launch_u(const Args &a, long long tokens, int rows, cudaStream_t st) {
  const int per = kThreads / G * U;
  norm_rope_kernel<DT, G, U, APPEND><<<dim3(static_cast<unsigned>(tokens), static_cast<unsigned>((rows + per - 1) / per)), kThreads, 0, st>>>(a);
  NB200_CHECK_CUDA(cudaGetLastError());
  return NB200_OK;
}
template <int DT, int G, bool APPEND> int launch_g(const Args &a, long long tokens, int rows, cudaStream_t st) {
  const int passes = (rows + kThreads / G - 1) / (kThreads / G);
  if (passes == 1 || tokens * passes <= 4 * 148) return launch_u<DT, G, 1, APPEND>(a, tokens, rows, st);
  if (passes == 2) return launch_u<DT, G, 2, APPEND>(a, tokens, rows, st);
  if (passes == 3) return launch_u<DT, G, 3, APPEND>(a, tokens, rows, st);
  return launch_u<DT, G, 4, APPEND>(a, tokens, rows, st);
}
template <int DT> int launch_dense(const Args &a, long long tokens, cudaStream_t st) {
  const int rows = a.Hq + a.Hkv;
  if (a.D <= 64) return launch_g<DT, 8, false>(a, tokens, rows, st);
  if (a.D <= 128) return launch_g<DT, 16, false>(a, tokens, rows, st);
  return launch_g<DT, 32, false>(a, tokens, rows, st);
}

int check_view(const char *who, const char *name, const void *p, const Strides &s, int size) {
  NB200_REQUIRE(aligned16(p), NB200_ERR_BAD_ARG, "%s: %s must be 16-byte aligned", who, name);
  NB200_REQUIRE(s.b * size % 16 == 0 && s.t * size % 16 == 0 && s.h * size % 16 == 0, NB200_ERR_BAD_ARG,
                "%s: the strides of %s must be multiples of 16 bytes", who, name);
  return NB200_OK;
}
int check_rotation(const char *who, int D, int rot, float eps) {
  NB200_REQUIRE(rot >= 16 && rot <= D && rot % 16 == 0, NB200_ERR_UNSUPPORTED,
                "%s: rot_dim = %d, a multiple of 16 from 16 to D = %d is needed", who, rot, D);
  NB200_REQUIRE(eps >= 0.f, NB200_ERR_BAD_ARG, "%s: eps must not be negative", who);
  return NB200_OK;
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" int nb200_qk_norm_rope(const void *q, const void *k, void *q_out, void *k_out, const int *positions,
                                  const float *inv_freq, const void *q_weight, const void *k_weight,
                                  const long long *strides, int B, int S, int Hq, int Hkv, int D, int rot_dim,
                                  int interleaved, float eps, int dtype, void *stream) {
  const char *who = "qk_norm_rope";
  NB200_REQUIRE(q && k && q_out && k_out && positions && inv_freq && strides, NB200_ERR_BAD_ARG, "%s: null pointer", who);
  NB200_REQUIRE(B > 0 && S > 0 && Hq > 0 && Hkv > 0 && D > 0, NB200_ERR_BAD_ARG, "%s: non-positive extent", who);
  NB200_REQUIRE(dtype == NB200_F16 || dtype == NB200_BF16 || dtype == NB200_F32, NB200_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  NB200_REQUIRE(D % 16 == 0 && D <= 256, NB200_ERR_UNSUPPORTED, "%s: D = %d, a multiple of 16 up to 256 is needed", who, D);
  NB200_REQUIRE(static_cast<long long>(B) * S < (1ll << 31), NB200_ERR_UNSUPPORTED, "%s: B * S does not fit 31 bits", who);
  NB200_REQUIRE(Hq <= 65535 && Hkv <= 65535, NB200_ERR_UNSUPPORTED, "%s: too many heads", who);
  int rc;
  if ((rc = check_rotation(who, D, rot_dim, eps)) != NB200_OK) return rc;
  Args a{};
  const int size = dtype == NB200_F32 ? 4 : 2;
  Strides *const views[4] = {&a.sq, &a.sk, &a.sqo, &a.sko};
  const void *const ptrs[4] = {q, k, q_out, k_out};
  const char *const names[4] = {"q", "k", "q_out", "k_out"};
  for (int i = 0; i < 4; ++i) {
    *views[i] = Strides{strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]};
    if ((rc = check_view(who, names[i], ptrs[i], *views[i], size)) != NB200_OK) return rc;
  }
  NB200_REQUIRE((!q_weight || aligned16(q_weight)) && (!k_weight || aligned16(k_weight)), NB200_ERR_BAD_ARG,
                "%s: the weights must be 16-byte aligned", who);
  a.q = q, a.k = k, a.q_out = q_out, a.k_out = k_out, a.wq = q_weight, a.wk = k_weight;
  a.inv_freq = inv_freq, a.positions = positions, a.positions_b = strides[12];
  a.S = S, a.Hq = Hq, a.Hkv = Hkv, a.D = D, a.rot = rot_dim, a.interleaved = interleaved, a.eps = eps, a.inv_d = 1.f / D;
  auto st = static_cast<cudaStream_t>(stream);
  const long long tokens = static_cast<long long>(B) * S;
  if (dtype == NB200_F16) return launch_dense<NB200_F16>(a, tokens, st);
  if (dtype == NB200_BF16) return launch_dense<NB200_BF16>(a, tokens, st);
  return launch_dense<NB200_F32>(a, tokens, st);
}

extern "C" int nb200_rope_append(const void *q, const void *k, const void *v, void *q_out, void *k_pages, void *v_pages,
                                 const int *block_table, const int *cu_seqlens, const int *seq_lens,
                                 const float *inv_freq, const void *q_weight, const void *k_weight,
                                 const long long *strides, int T, int B, int Hq, int Hkv, int num_pages, int max_pages,
                                 int page_size, int D, int rot_dim, int interleaved, float eps, int dtype, int *status,
                                 void *stream) {
  const char *who = "rope_append";
  NB200_REQUIRE(k && v && k_pages && v_pages && block_table && cu_seqlens && seq_lens && inv_freq && strides,
                NB200_ERR_BAD_ARG, "%s: null pointer", who);
  NB200_REQUIRE(T > 0 && B > 0 && Hkv > 0 && num_pages > 0 && max_pages > 0 && D > 0 && Hq >= 0, NB200_ERR_BAD_ARG,
                "%s: non-positive extent", who);
  NB200_REQUIRE(Hq == 0 || (q && q_out), NB200_ERR_BAD_ARG, "%s: null pointer", who);
  NB200_REQUIRE(dtype == NB200_F16 || dtype == NB200_BF16, NB200_ERR_UNSUPPORTED, "%s: dtype %d (f16 and bf16 only)", who, dtype);
  NB200_REQUIRE(D == kCacheD, NB200_ERR_UNSUPPORTED, "%s: D = %d, only 128 is implemented", who, D);
  NB200_REQUIRE(page_size == kPageRows, NB200_ERR_UNSUPPORTED, "%s: page_size = %d, only %d rows per page is implemented", who,
                page_size, kPageRows);
  NB200_REQUIRE(max_pages <= (0x7fffffff / kPageRows), NB200_ERR_UNSUPPORTED, "%s: max_pages * page_size does not fit 31 bits", who);
  NB200_REQUIRE(Hq <= 65535 && Hkv <= 65535, NB200_ERR_UNSUPPORTED, "%s: too many heads", who);
  int rc;
  if ((rc = check_rotation(who, D, rot_dim, eps)) != NB200_OK) return rc;
  Args a{};
  Strides *const views[4] = {&a.sq, &a.sk, &a.sv, &a.sqo};
  const void *const ptrs[4] = {q, k, v, q_out};
  const char *const names[4] = {"q", "k", "v", "q_out"};
  for (int i = 0; i < 4; ++i) {
    if (Hq == 0 && (i == 0 || i == 3)) continue;
    *views[i] = Strides{0, strides[2 * i], strides[2 * i + 1]};
    if ((rc = check_view(who, names[i], ptrs[i], *views[i], 2)) != NB200_OK) return rc;
  }
  NB200_REQUIRE(aligned16(k_pages) && aligned16(v_pages), NB200_ERR_BAD_ARG, "%s: the page pools must be 16-byte aligned", who);
  NB200_REQUIRE((!q_weight || aligned16(q_weight)) && (!k_weight || aligned16(k_weight)), NB200_ERR_BAD_ARG,
                "%s: the weights must be 16-byte aligned", who);
  a.q = q, a.k = k, a.v = v, a.q_out = q_out, a.wq = q_weight, a.wk = k_weight, a.inv_freq = inv_freq;
  a.S = T, a.Hq = Hq, a.Hkv = Hkv, a.D = D, a.rot = rot_dim, a.interleaved = interleaved, a.eps = eps, a.inv_d = 1.f / D;
  a.k_pages = k_pages, a.v_pages = v_pages, a.block_table = block_table, a.cu_seqlens = cu_seqlens, a.seq_lens = seq_lens;
  a.B = B, a.num_pages = num_pages, a.max_pages = max_pages, a.status = status;
  auto st = static_cast<cudaStream_t>(stream);
  if (dtype == NB200_F16) return launch_g<NB200_F16, 16, true>(a, T, Hq + 2 * Hkv, st);
  return launch_g<NB200_BF16, 16, true>(a, T, Hq + 2 * Hkv, st);
}
