// Attention of the new tokens of a ragged batch over the paged KV cache.
//
// Token t of sequence b (cu_seqlens[b] <= t < cu_seqlens[b+1]) sits at position p = seq_lens[b] - cu_seqlens[b+1] + t and
// sees the cached rows j <= p, its own among them:  out[t, h] = sum_j softmax_j(q[t, h] . k_j * scale) v_j, query head h
// reading kv head h / (Hq / Hkv).  One warp per (token, query head), one pass over the rows with the running maximum and
// sum of the softmax in fp32.
#include "nb200_common.cuh"

namespace nb200 {
namespace {

constexpr int kPageRows = 64;
constexpr int kD = 128;
constexpr int kErrTable = 22;

struct Args {
  const void *q, *k_pages, *v_pages;
  void *out;
  const int *block_table, *cu_seqlens, *seq_lens;
  long long q_t, q_h, out_t, out_h;
  int T, B, Hq, Hkv, num_pages, max_pages;
  float scale_log2;
  int *status;
};

template <int DT> __global__ void __launch_bounds__(32) attn_paged_kernel(const Args a) {
  const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  int below = 0;
  for (int i = lane; i <= a.B; i += 32) below += a.cu_seqlens[i] <= t;
  const int b = __reduce_add_sync(0xffffffffu, below) - 1;
  if (b < 0 || b >= a.B || t < a.cu_seqlens[b] || t >= a.cu_seqlens[b + 1]) return;
  const long long p = static_cast<long long>(a.seq_lens[b]) - a.cu_seqlens[b + 1] + t;
  const long long last = min(p, min(static_cast<long long>(a.seq_lens[b]), static_cast<long long>(a.max_pages) * kPageRows) - 1);
  float2 q01 = unpack2<DT>(reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.q) + t * a.q_t + h * a.q_h)[lane].x);
  float2 q23 = unpack2<DT>(reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.q) + t * a.q_t + h * a.q_h)[lane].y);
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  const int kv = h / (a.Hq / a.Hkv);
  bool bad = false;
  for (long long j = 0; j <= last; ++j) {
    const int page = a.block_table[static_cast<long long>(b) * a.max_pages + j / kPageRows];
    if (page < 0 || page >= a.num_pages) {
      if (a.status && lane == 0 && atomicCAS(a.status, 0, kErrTable) == 0) {
        a.status[1] = static_cast<int>(blockIdx.x);
        a.status[2] = page;
        a.status[3] = lane;
      }
      bad = true;
      break;
    }
    const long long row = ((static_cast<long long>(page) * a.Hkv + kv) * kPageRows + j % kPageRows) * kD;
    const uint2 kw = reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.k_pages) + row)[lane];
    const uint2 vw = reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.v_pages) + row)[lane];
    const float2 k01 = unpack2<DT>(kw.x), k23 = unpack2<DT>(kw.y), v01 = unpack2<DT>(vw.x), v23 = unpack2<DT>(vw.y);
    float x = q01.x * k01.x + q01.y * k01.y + q23.x * k23.x + q23.y * k23.y;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
    x *= a.scale_log2;
    const float m_new = fmaxf(m, x), f = m == m_new ? 1.f : ex2(m - m_new), w = ex2(x - m_new);
    m = m_new;
    l = l * f + w;
    o[0] = o[0] * f + w * v01.x;
    o[1] = o[1] * f + w * v01.y;
    o[2] = o[2] * f + w * v23.x;
    o[3] = o[3] * f + w * v23.y;
  }
  const float inv = bad ? __int_as_float(0x7fffffff) : (l == 0.f ? 0.f : 1.f / l);   // a row that sees nothing is 0
  reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + t * a.out_t + h * a.out_h)[lane] =
      make_uint2(pack2<DT>(o[0] * inv, o[1] * inv), pack2<DT>(o[2] * inv, o[3] * inv));
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" size_t nb200_attn_paged_workspace_bytes(void) { return 160 * 2 * 128 * (kD + 2) * sizeof(float) + 160 * 64; }

extern "C" int nb200_attn_paged(const void *q, const void *k_pages, const void *v_pages, const int *block_table,
                                const int *cu_seqlens, const int *seq_lens, void *workspace, void *out,
                                const long long *strides, int T, int B, int Hq, int Hkv, int num_pages, int max_pages,
                                int page_size, int D, int dtype, float scale_log2, int *status, void *stream) {
  const char *who = "attn_paged";
  NB200_REQUIRE(q && k_pages && v_pages && block_table && cu_seqlens && seq_lens && workspace && out && strides,
                NB200_ERR_BAD_ARG, "%s: null pointer", who);
  NB200_REQUIRE(T > 0 && B > 0 && Hq > 0 && Hkv > 0 && num_pages > 0 && max_pages > 0 && D > 0, NB200_ERR_BAD_ARG,
                "%s: non-positive extent", who);
  NB200_REQUIRE(scale_log2 > 0.f, NB200_ERR_BAD_ARG, "%s: scale_log2 must be positive", who);
  NB200_REQUIRE(dtype == NB200_F16 || dtype == NB200_BF16, NB200_ERR_UNSUPPORTED, "%s: dtype %d (f16 and bf16 only)", who, dtype);
  NB200_REQUIRE(D == kD, NB200_ERR_UNSUPPORTED, "%s: D = %d, only 128 is implemented", who, D);
  NB200_REQUIRE(page_size == kPageRows, NB200_ERR_UNSUPPORTED, "%s: page_size = %d, only %d rows per page is implemented", who,
                page_size, kPageRows);
  NB200_REQUIRE(Hq % Hkv == 0, NB200_ERR_UNSUPPORTED, "%s: Hq %% Hkv != 0", who);
  NB200_REQUIRE(Hq / Hkv <= 128, NB200_ERR_UNSUPPORTED, "%s: more than 128 query heads per kv head", who);
  NB200_REQUIRE(Hq <= 65535, NB200_ERR_UNSUPPORTED, "%s: too many heads", who);
  NB200_REQUIRE(max_pages <= (0x7fffffff / kPageRows), NB200_ERR_UNSUPPORTED, "%s: max_pages * page_size does not fit 31 bits", who);
  NB200_REQUIRE(static_cast<long long>(num_pages) * Hkv < (1ll << 31), NB200_ERR_UNSUPPORTED,
                "%s: num_pages * Hkv does not fit 31 bits", who);
  NB200_REQUIRE(aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(out) && aligned16(workspace),
                NB200_ERR_BAD_ARG, "%s: q, out, the page pools and the workspace must be 16-byte aligned", who);
  for (int i = 0; i < 4; ++i)
    NB200_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0, NB200_ERR_BAD_ARG,
                  "%s: the strides of q and out must be multiples of 16 bytes", who);
  Args a{q, k_pages, v_pages, out, block_table, cu_seqlens, seq_lens, strides[0], strides[1], strides[2], strides[3],
         T, B, Hq, Hkv, num_pages, max_pages, scale_log2, status};
  auto st = static_cast<cudaStream_t>(stream);
  if (dtype == NB200_BF16)
    attn_paged_kernel<NB200_BF16><<<dim3(T, Hq), 32, 0, st>>>(a);
  else
    attn_paged_kernel<NB200_F16><<<dim3(T, Hq), 32, 0, st>>>(a);
  NB200_CHECK_CUDA(cudaGetLastError());
  return NB200_OK;
}
