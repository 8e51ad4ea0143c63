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
// A warp takes a token, or part of its rows where there are few tokens.  A row is read by G lanes, and lane u holds the
// elements {4u .. 4u+3} and {rot/2 + 4u ..} (halves) or {8u .. 8u+7} (neighbours): both elements of a pair and the same
// four angles either way, so a rotation needs no shuffle, and the sines and cosines, which a lane computes two of, are
// read from shared memory once for all the rows of the token.  No barrier wider than a warp; four rows' loads are in
// flight at a time, the first four while the token's sequence, page and angles are looked up.
//
// What bounds it is HBM: 8 x 4096 tokens of 32 / 32 heads with norms in 185 us alone from idle clocks (5.8 TB/s, where a
// plain copy of the same bytes takes 168), 192 to 199 one call after the other (5.4 TB/s); in fp32 335 us (6.4 TB/s).  An
// append of 2 x 8192 tokens of 32 / 8 heads takes 74 us alone (5.4 TB/s), 76 one after the other (5.3); builds that skipped the
// look-up of the page, and the angles, took 2 and 1 us less.  Small calls are bound by the launch: 2.5 to 3.4 us on the
// GPU, 3.3 to 5 us of host time.
#include "nb200_common.cuh"

namespace nb200 {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;             // rows of a lane in flight
constexpr int kMaxHalf = 128;          // rot <= 256
constexpr int kPageRows = 64;
constexpr int kCacheD = 128;

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

// Four consecutive elements of a row as they are stored: 8 bytes, or 16 in fp32.
template <int DT> struct Piece {
  using type = uint2;
};
template <> struct Piece<NB200_F32> {
  using type = uint4;
};
template <int DT> using piece_t = typename Piece<DT>::type;
template <int DT> __device__ __forceinline__ piece_t<DT> load_piece(const void *base, long long elem) {
  return *reinterpret_cast<const piece_t<DT> *>(static_cast<const char *>(base) + elem * (DT == NB200_F32 ? 4 : 2));
}
template <int DT> __device__ __forceinline__ void store_piece(void *base, long long elem, piece_t<DT> x) {
  *reinterpret_cast<piece_t<DT> *>(static_cast<char *>(base) + elem * (DT == NB200_F32 ? 4 : 2)) = x;
}
template <int DT> __device__ __forceinline__ void to_float(piece_t<DT> r, float *y) {
  if constexpr (DT == NB200_F32) {
    y[0] = __uint_as_float(r.x), y[1] = __uint_as_float(r.y), y[2] = __uint_as_float(r.z), y[3] = __uint_as_float(r.w);
  } else {
    const float2 f = unpack2<DT>(r.x), g = unpack2<DT>(r.y);
    y[0] = f.x, y[1] = f.y, y[2] = g.x, y[3] = g.y;
  }
}
template <int DT> __device__ __forceinline__ piece_t<DT> from_float(const float *y) {
  if constexpr (DT == NB200_F32)
    return make_uint4(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3]));
  else
    return make_uint2(pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3]));
}

__device__ __forceinline__ void report(int *status, int code, int detail, int detail2) {
  status_record(status, code, static_cast<int>(blockIdx.x), detail, detail2);
}

// Sequence whose tokens include row t, or -1: one before the first entry of cu_seqlens [B + 1] above t, found 32 ways at
// a time by the whole warp.
__device__ __forceinline__ int sequence_of(const int *cu, int B, int t, int lane) {
  int lo = 0, n = B + 1;                                  // entries [0, lo) are <= t; the first above t is in [lo, lo + n]
  while (n > 0) {
    const int step = (n + 31) / 32, i = lo + lane * step;
    const int below = __popc(__ballot_sync(0xffffffffu, lane * step < n && cu[min(i, B)] <= t));
    if (below == 0) break;                                // entry lo is above t
    const int probe = lo + (below - 1) * step;            // the last probe that is <= t
    n = min(step - 1, lo + n - probe - 1);
    lo = probe + 1;
  }
  return lo - 1 < B ? lo - 1 : -1;
}

// Rows of a token: Hq queries, then Hkv keys, then (append) Hkv values.  Warp `unit` of the grid takes rows
// [chunk * per, chunk * per + per) of a token, 32 / G at a time.
//
// What bounds it beside HBM is the issue rate, so the arithmetic is on packed pairs of fp32, the weights are converted
// once per token, and pointers advance by adding: 184 warp instructions per 32 / G rows went down to about 70.
template <int DT, int G, bool APPEND, bool NEIGHBOURS>
__global__ void __launch_bounds__(kThreads, DT == NB200_F32 ? 5 : 7) norm_rope_kernel(const Args a, const unsigned units, const unsigned chunks, const int per) {
  constexpr int kRows = 32 / G;
  constexpr int kSize = DT == NB200_F32 ? 4 : 2;
  __shared__ float4 turns[kWarps][kMaxHalf / 2];          // (cos, sin) of the token's angles, two to a word
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");        // launched as a programmatic dependent
  const unsigned unit = blockIdx.x * kWarps + warp;
  if (unit >= units) return;
  const int t = static_cast<int>(unit / chunks), chunk = static_cast<int>(unit % chunks);
  const int u = lane % G, sub = lane / G;
  const bool in_row = u * 8 < a.D;
  const bool turned = u * 8 < a.rot;
  // byte offsets of the lane's two pieces
  const int e0 = (turned && !NEIGHBOURS ? 4 * u : 8 * u) * kSize, e1 = (turned && !NEIGHBOURS ? a.rot / 2 + 4 * u : 8 * u + 4) * kSize;
  const long long bt = APPEND ? 0 : t / a.S, st = APPEND ? t : t % a.S;

  // The first rows' loads are in flight while the token's place and angles are looked up.
  const int row_lo = chunk * per, row_hi = row_lo + per;
  int kind = row_lo < a.Hq ? 0 : 1, lo = 0, hi = 0;        // queries, keys; the warp's rows of that kind
  const char *src = nullptr;
  long long src_step = 0;
  piece_t<DT> x0[kUnroll], x1[kUnroll];
  auto open = [&]() {
    const int begin = kind ? a.Hq : 0;
    lo = max(row_lo, begin);
    hi = min(row_hi, kind ? a.Hq + a.Hkv : a.Hq);
    const Strides &in = kind ? a.sk : a.sq;
    src = static_cast<const char *>(kind ? a.k : a.q) + (bt * in.b + st * in.t + (lo - begin + sub) * in.h) * kSize + e0;
    src_step = in.h * kRows * kSize;
  };
  auto fetch = [&](int row0) {
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      x0[i] = x1[i] = piece_t<DT>{};
      if (in_row && row0 + i * kRows + sub < hi) {
        x0[i] = load_piece<DT>(src, 0);
        x1[i] = load_piece<DT>(src + (e1 - e0), 0);
      }
      src += src_step;
    }
  };
  open();
  fetch(lo);

  int pos = 0;
  long long slot_base = 0;                                // element offset of (page, head 0, row) in the pools
  if constexpr (APPEND) {
    const int b = sequence_of(a.cu_seqlens, a.B, t, lane);
    if (b < 0) return;                                    // a row of no sequence: left as it was
    const int first = a.cu_seqlens[b], end = a.cu_seqlens[b + 1];
    if (t < first || t >= end) return;                    // cu_seqlens is not a running sum
    const long long p = static_cast<long long>(a.seq_lens[b]) - end + t;
    if (p < 0 || p >= static_cast<long long>(a.max_pages) * kPageRows) {
      if (lane == 0 && chunk == 0) report(a.status, kStatusNoSlot, t, static_cast<int>(p));
      return;
    }
    pos = static_cast<int>(p);
    const int page = a.block_table[static_cast<long long>(b) * a.max_pages + pos / kPageRows];
    if (page < 0 || page >= a.num_pages) {
      if (lane == 0 && chunk == 0) report(a.status, kStatusBadPage, page, 0);
      return;
    }
    slot_base = (static_cast<long long>(page) * a.Hkv * kPageRows + pos % kPageRows) * kCacheD;
  } else {
    pos = a.positions[bt * a.positions_b + st];
  }

  if (row_lo < a.Hq + a.Hkv) {                            // else values alone
    for (int i = lane; i < a.rot / 2; i += 32) {
      const double x = static_cast<double>(pos) * static_cast<double>(a.inv_freq[i]) * 0.15915494309189535;   // 1 / 2 pi
      float s, c;
      sincospif(2.f * static_cast<float>(x - rint(x)), &s, &c);
      reinterpret_cast<float2 *>(turns[warp])[i] = make_float2(c, s);
    }
  }
  __syncwarp();
  // cos, sin and -sin of the angles 4u .. 4u + 3, in pairs
  uint64_t c2[2], s2[2], n2[2];
  {
    float4 x = make_float4(1.f, 0.f, 1.f, 0.f), y = x;
    if (turned) x = turns[warp][2 * u], y = turns[warp][2 * u + 1];
    c2[0] = f2_pack(x.x, x.z), s2[0] = f2_pack(x.y, x.w), n2[0] = f2_pack(-x.y, -x.w);
    c2[1] = f2_pack(y.x, y.z), s2[1] = f2_pack(y.y, y.w), n2[1] = f2_pack(-y.y, -y.w);
  }

  // queries, then keys
#pragma unroll 1
  while (true) {
    const int begin = kind ? a.Hq : 0;
    char *dst;
    long long dst_step;
    if (APPEND && kind) {
      dst = static_cast<char *>(a.k_pages) + (slot_base + static_cast<long long>(lo - begin + sub) * (kPageRows * kCacheD)) * kSize + e0;
      dst_step = static_cast<long long>(kPageRows) * kCacheD * kRows * kSize;
    } else {
      const Strides to = kind ? a.sko : a.sqo;
      dst = static_cast<char *>(kind ? a.k_out : a.q_out) + (bt * to.b + st * to.t + (lo - begin + sub) * to.h) * kSize + e0;
      dst_step = to.h * kRows * kSize;
    }
    const void *w = kind ? a.wk : a.wq;
    // element pairs: f[0..1] are the first elements of the lane's four pairs, f[2..3] the second ones
    auto unpack = [&](piece_t<DT> p0, piece_t<DT> p1, uint64_t (&f)[4]) {
      float y[8];
      to_float<DT>(p0, y);
      to_float<DT>(p1, y + 4);
      if constexpr (NEIGHBOURS) {
        f[0] = f2_pack(y[0], y[2]), f[1] = f2_pack(y[4], y[6]), f[2] = f2_pack(y[1], y[3]), f[3] = f2_pack(y[5], y[7]);
      } else {
        f[0] = f2_pack(y[0], y[1]), f[1] = f2_pack(y[2], y[3]), f[2] = f2_pack(y[4], y[5]), f[3] = f2_pack(y[6], y[7]);
      }
    };
    uint64_t g[4] = {};
    if (w && in_row)
      unpack(load_piece<DT>(static_cast<const char *>(w) + e0, 0), load_piece<DT>(static_cast<const char *>(w) + e1, 0), g);
#pragma unroll 1
    for (int row0 = lo; row0 < hi; row0 += kUnroll * kRows) {
      if (row0 > lo) fetch(row0);
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        if (row0 + i * kRows >= hi) break;                // the same for the whole warp
        uint64_t f[4];
        unpack(x0[i], x1[i], f);
        if (w) {
          uint64_t sq = f2_mul(f[0], f[0]);
#pragma unroll
          for (int e = 1; e < 4; ++e) sq = f2_fma(f[e], f[e], sq);
          const float2 both = f2_unpack(sq);
          float ss = both.x + both.y;
#pragma unroll
          for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float r = rsqrtf(fmaf(ss, a.inv_d, a.eps));
          const uint64_t r2 = f2_pack(r, r);
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] = f2_mul(f2_mul(f[e], r2), g[e]);
        }
        if (turned) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint64_t y1 = f[e], y2 = f[e + 2];
            f[e] = f2_fma(y2, n2[e], f2_mul(y1, c2[e]));
            f[e + 2] = f2_fma(y1, s2[e], f2_mul(y2, c2[e]));
          }
        }
        float y[8];
        {
          const float2 p = f2_unpack(f[0]), q = f2_unpack(f[1]), v = f2_unpack(f[2]), z = f2_unpack(f[3]);
          if constexpr (NEIGHBOURS) {
            y[0] = p.x, y[2] = p.y, y[4] = q.x, y[6] = q.y, y[1] = v.x, y[3] = v.y, y[5] = z.x, y[7] = z.y;
          } else {
            y[0] = p.x, y[1] = p.y, y[2] = q.x, y[3] = q.y, y[4] = v.x, y[5] = v.y, y[6] = z.x, y[7] = z.y;
          }
        }
        if (in_row && row0 + i * kRows + sub < hi) {
          store_piece<DT>(dst, 0, from_float<DT>(y));
          store_piece<DT>(dst + (e1 - e0), 0, from_float<DT>(y + 4));
        }
        dst += dst_step;
      }
    }
    if (kind == 1) break;
    kind = 1;
    open();
    fetch(lo);
  }
  if constexpr (APPEND) {                                 // values: copied as they are
    const int begin = a.Hq + a.Hkv, lo = max(row_lo, begin), hi = min(row_hi, begin + a.Hkv);
    const char *src = static_cast<const char *>(a.v) + (st * a.sv.t + (lo - begin + sub) * a.sv.h) * 2 + u * 16;
    char *dst = static_cast<char *>(a.v_pages) + (slot_base + static_cast<long long>(lo - begin + sub) * (kPageRows * kCacheD)) * 2 + u * 16;
#pragma unroll 4
    for (int row = lo + sub; row < hi; row += kRows) {
      *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(src);
      src += a.sv.h * kRows * 2;
      dst += static_cast<long long>(kPageRows) * kCacheD * kRows * 2;
    }
  }
}

// A warp does all the rows of a token where the tokens alone fill the SMs' warps; with fewer tokens their rows are dealt
// out, down to one pass per warp, which then computes the token's angles again.
template <int DT, int G, bool APPEND> int launch_g(const Args &a, long long tokens, int rows, cudaStream_t st) {
  constexpr int kResident = 148 * (DT == NB200_F32 ? 5 : 7) * kWarps, kRows = 32 / G;   // blocks to an SM by the launch bounds
  const int passes = (rows + kRows - 1) / kRows;
  long long per = (tokens * passes + kResident - 1) / kResident;
  per = per < 1 ? 1 : (per >= passes ? passes : per);
  if (per > kUnroll) per = (per + kUnroll - 1) / kUnroll * kUnroll;
  const long long chunks = (passes + per - 1) / per, units = tokens * chunks;
  NB200_REQUIRE(units < (1ll << 31), NB200_ERR_UNSUPPORTED, "norm and rotation: too many rows");
  const unsigned blocks = static_cast<unsigned>((units + kWarps - 1) / kWarps);
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;   // the launch overlaps the end of the kernel before
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const unsigned n = static_cast<unsigned>(units), c = static_cast<unsigned>(chunks);
  NB200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, a.interleaved ? norm_rope_kernel<DT, G, APPEND, true> : norm_rope_kernel<DT, G, APPEND, false>,
                                      a, n, c, static_cast<int>(per) * kRows));
  return NB200_OK;
}
template <int DT> int launch_dense(const Args &a, long long tokens, cudaStream_t st) {
  const int rows = a.Hq + a.Hkv;
  if (a.D <= 64) return launch_g<DT, 8, false>(a, tokens, rows, st);
  if (a.D <= 128) return launch_g<DT, 16, false>(a, tokens, rows, st);
  return launch_g<DT, 32, false>(a, tokens, rows, st);
}

int check_view(const char *who, const char *name, const void *p, const Strides &s, int B, int S, int size) {
  auto fits = [&](int extent, long long stride) { return extent == 1 || stride * size % 16 == 0; };   // one that is taken
  NB200_REQUIRE(aligned16(p), NB200_ERR_BAD_ARG, "%s: %s must be 16-byte aligned", who, name);
  NB200_REQUIRE(fits(B, s.b) && fits(S, s.t) && s.h * size % 16 == 0, NB200_ERR_BAD_ARG,
                "%s: the strides of %s must be multiples of 16 bytes", who, name);
  return NB200_OK;
}
// An output's rows must not lie over one another, as those of an expanded tensor do.
int check_rows_apart(const char *who, const char *name, const Strides &s, int B, int S, int H, int D) {
  auto apart = [&](int extent, long long stride) { return extent == 1 || stride >= D || stride <= -D; };
  NB200_REQUIRE(apart(B, s.b) && apart(S, s.t) && apart(H, s.h), NB200_ERR_BAD_ARG,
                "%s: the strides of %s must be at least a row", who, name);
  NB200_REQUIRE(rows_apart(D, {B, S, H}, {s.b, s.t, s.h}), NB200_ERR_BAD_ARG, "%s: the rows of %s must lie apart", who, name);
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
    const int H = i % 2 == 0 ? Hq : Hkv;
    if ((rc = check_view(who, names[i], ptrs[i], *views[i], B, S, size)) != NB200_OK) return rc;
    if (i >= 2 && (rc = check_rows_apart(who, names[i], *views[i], B, S, H, D)) != NB200_OK) return rc;
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
    if ((rc = check_view(who, names[i], ptrs[i], *views[i], 1, T, 2)) != NB200_OK) return rc;
    if (i == 3 && (rc = check_rows_apart(who, names[i], *views[i], 1, T, Hq, D)) != NB200_OK) return rc;
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
