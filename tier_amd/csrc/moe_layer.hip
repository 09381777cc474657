// moe_layer.hip -- a routed layer of a few tokens over int8 experts: gate and up, the gate's
// activation, down, and the weighted sum of a token's experts.  No reference function (the
// reference refuses MoE models, arch.py:158-159).
//
//   g, u = int8 products of x with an expert's gate and up rows (tm_i8.h: exact sums, fp32 scales)
//   h = fp32(silu(g) u), in 64 bits, rounded once
//   hq = codes of h's row, scale max|h| / 127, as tiermm_i8_quant makes them
//   out[t] = sum_j weights[t][j] * (int8 product of hq with the down rows), in j order in fp32
//
// 64 bits for the gate: h is then the same fp32 number whatever exp does in its last bits, and its
// codes with it.
#include "tm_i8.h"

namespace tiermm {
namespace {

constexpr int kTokens = TIERMM_MOE_LAYER_TOKENS, kTopk = TIERMM_MOE_LAYER_TOPK, kPairs = kTokens * kTopk;

struct LayerArgs {
  const uint8_t *X, *Wg, *Wd;        // codes: T rows, E * 2F rows (gate, then up), E * K rows
  const float *sx, *sg, *sd, *weights;
  const int32_t* ids;
  float* h;                          // [P][F]
  uint32_t* top;                     // [P][tiles of F]: largest |h|, as bits
  float* y;                          // [P][K]
  uint8_t* out;
  size_t rbx, rbg, rbd, ldo;         // bytes
  int T, topk, P, E, K, F, nk, nf;   // nk, nf: 64-byte steps of x's and h's rows
  int by_pair;                       // slots are pairs (fewer than experts): the first of an expert's acts
};

// The pairs of this workgroup's expert, in order, into list; returns their number (0: nothing to do).
// An id outside [0, E) is a dropped pair.
__device__ __forceinline__ int find_pairs(const LayerArgs& a, int slot, int& e, uint16_t* list) {
  const int lane = threadIdx.x & 63;
  e = a.by_pair ? a.ids[slot] : slot;
  if ((uint32_t)e >= (uint32_t)a.E) return 0;
  int n = 0;
  for (int p0 = 0; p0 < a.P; p0 += 64) {
    const int p = p0 + lane;
    const uint64_t hit = __ballot(p < a.P && a.ids[min(p, a.P - 1)] == e);
    if (a.by_pair && hit && n == 0 && p0 + __ffsll((unsigned long long)hit) - 1 < slot) return 0;
    // (every wave writes the same list)
    if (hit >> lane & 1) list[n + __popcll(hit & ((1ull << lane) - 1))] = (uint16_t)p;
    n += __popcll(hit);
  }
  return n;
}

// Tile of 16 rows of the gate and the same 16 of up, times the expert's tokens, 16 at a time; the
// four waves share K.
__global__ __launch_bounds__(256) void moe_gate_up_kernel(const LayerArgs a) {
  __shared__ uint16_t list[kPairs];
  __shared__ __attribute__((aligned(16))) int32_t sums[4][2][16][20];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
  int e;
  const int n = find_pairs(a, blockIdx.y, e, list);
  if (n == 0) return;
  const int f0 = blockIdx.x * 16, fr = min(f0 + r, a.F - 1);
  const uint8_t* wg = a.Wg + ((size_t)e * 2 * a.F + fr) * a.rbg + 16 * g;
  const uint8_t* wu = wg + (size_t)a.F * a.rbg;
  __syncthreads();
  const int s0 = a.nk * wave / 4, s1 = a.nk * (wave + 1) / 4;
  for (int base = 0; base < n; base += 16) {
    const uint8_t* x = a.X + (size_t)(list[min(base + r, n - 1)] / a.topk) * a.rbx + 16 * g;
    i32x4 ag = {0, 0, 0, 0}, au = {0, 0, 0, 0};
    for (int s = s0; s < s1; ++s) {
      const i32x4 b = *(const i32x4*)(x + (size_t)s * 64);
      ag = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4*)(wg + (size_t)s * 64), b, ag, 0, 0, 0);
      au = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4*)(wu + (size_t)s * 64), b, au, 0, 0, 0);
    }
    *(i32x4*)&sums[wave][0][r][4 * g] = ag;
    *(i32x4*)&sums[wave][1][r][4 * g] = au;
    __syncthreads();
    const int c = tid >> 4, f = tid & 15;
    int sg = 0, su = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      sg += sums[w][0][c][f];
      su += sums[w][1][c][f];
    }
    if (base + c < n) {
      const int p = list[base + c];
      uint32_t top = 0;
      if (f0 + f < a.F) {
        const size_t ch = (size_t)e * 2 * a.F + f0 + f;
        const float sx = a.sx[p / a.topk];
        const double gate = scaled(sg, sx, a.sg[ch], 0.f), up = scaled(su, sx, a.sg[ch + a.F], 0.f);
        const float h = (float)(gate / (1. + exp(-gate)) * up);
        a.h[(size_t)p * a.F + f0 + f] = h;
        top = __float_as_uint(h) & 0x7fffffffu;
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 16));
      if (f == 0) a.top[(size_t)p * gridDim.x + blockIdx.x] = top;
    }
    __syncthreads();
  }
}

// Tile of 16 rows of the down weight times the codes of h's rows, which each wave makes of its own
// share of K.
__global__ __launch_bounds__(256) void moe_down_kernel(const LayerArgs a) {
  __shared__ uint16_t list[kPairs];
  __shared__ __attribute__((aligned(16))) int32_t sums[4][16][20];
  __shared__ RowScale scale[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
  int e;
  const int n = find_pairs(a, blockIdx.y, e, list);
  if (n == 0) return;
  const int k0 = blockIdx.x * 16, kr = min(k0 + r, a.K - 1), nt = (a.F + 15) / 16;
  const uint8_t* w = a.Wd + ((size_t)e * a.K + kr) * a.rbd + 16 * g;
  __syncthreads();
  const int s0 = a.nf * wave / 4, s1 = a.nf * (wave + 1) / 4;
  for (int base = 0; base < n; base += 16) {
    const int c = tid >> 4, i0 = tid & 15;
    uint32_t top = 0;
    for (int i = i0; i < nt; i += 16) top = max(top, a.top[(size_t)list[min(base + c, n - 1)] * nt + i]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 16));
    if (i0 == 0) scale[c] = row_scale_of(top);
    __syncthreads();
    const RowScale rs = scale[r];
    const float* h = a.h + (size_t)list[min(base + r, n - 1)] * a.F;
    i32x4 acc = {0, 0, 0, 0};
    for (int s = s0; s < s1; ++s) {
      i32x4 b;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int f = s * 64 + 16 * g + 4 * q + i;
          v[i] = f < a.F ? h[f] : 0.f;
        }
        b[q] = (int)codes4(v, rs);
      }
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4*)(w + (size_t)s * 64), b, acc, 0, 0, 0);
    }
    *(i32x4*)&sums[wave][r][4 * g] = acc;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int v = 0; v < 4; ++v) sum += sums[v][c][i0];
    if (base + c < n && k0 + i0 < a.K)
      a.y[(size_t)list[base + c] * a.K + k0 + i0] = scaled(sum, scale[c].sc, a.sd[(size_t)e * a.K + k0 + i0], 0.f);
    __syncthreads();
  }
}

// out[t] = sum_j weights[t][j] y[t][j], dropped pairs skipped.
template <int YT>
__global__ __launch_bounds__(256) void moe_layer_sum_kernel(const LayerArgs a) {
  using Y = Rows<YT>;
  const int t = blockIdx.x, c = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (c >= a.K) return;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < a.topk; ++j) {
    const int p = t * a.topk + j;
    if ((uint32_t)a.ids[p] >= (uint32_t)a.E) continue;
    const float w = a.weights[p];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fmaf(w, c + i < a.K ? a.y[(size_t)p * a.K + c + i] : 0.f, acc[i]);
  }
  Y::put4(a.out + (size_t)t * a.ldo + (size_t)c * Y::ES, acc, min(4, a.K - c));
}

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

}  // namespace
}  // namespace tiermm

using namespace tiermm;

extern "C" {

size_t tiermm_moe_i8_layer_ws_bytes(int T, int topk, int K, int F) {
  if (T < 1 || topk < 1 || K < 1 || F < 1 || T > kTokens || topk > kTopk || K > kMaxK || F > kMaxK) return 0;
  const size_t P = (size_t)T * topk;
  return align16(P * F * 4) + align16(P * K * 4) + align16(P * ((F + 15) / 16) * 4);
}

int tiermm_moe_i8_layer(const int8_t* Xq, size_t rbx, const float* sx, const int32_t* expert_ids, const float* weights,
                        const int8_t* Wgu, size_t rbg, const float* sgu, const int8_t* Wd, size_t rbd, const float* sd,
                        void* out, int otype, size_t ldo, int T, int topk, int n_experts, int K, int F, void* ws,
                        size_t ws_bytes, tiermm_stream_t stream) {
  const char* who = "tiermm_moe_i8_layer";
  if (T < 0 || topk < 0 || n_experts < 1 || K < 1 || F < 1) return set_error(TIERMM_EINVAL, "%s: bad size", who);
  if (T > kTokens || topk > kTopk)
    return set_error(TIERMM_UNSUPPORTED, "%s: %d tokens of %d experts, at most %d of %d", who, T, topk, kTokens, kTopk);
  if (n_experts > TIERMM_MOE_MAX_EXPERTS)
    return set_error(TIERMM_UNSUPPORTED, "%s: %d experts, at most %d", who, n_experts, TIERMM_MOE_MAX_EXPERTS);
  if (K > kMaxK || F > kMaxK) return set_error(TIERMM_UNSUPPORTED, "%s: K = %d, F = %d, at most %d", who, K, F, kMaxK);
  const int es = row_elem_bytes(otype);
  if (!es) return set_error(TIERMM_UNSUPPORTED, "%s: output of type %d", who, otype);
  if (bad_stride(ldo, K)) return set_error(TIERMM_EINVAL, "%s: row stride below %d or past 2^40", who, K);
  if (T == 0) return TIERMM_OK;
  if (!out || misaligned(out, es)) return set_error(TIERMM_EINVAL, "%s: null or misaligned output", who);
  const struct { const void* p; size_t rb; int K; } rows[] = {{Xq, rbx, K}, {Wgu, rbg, K}, {Wd, rbd, F}};
  for (const auto& r : rows)
    if (topk && (!r.p || misaligned(r.p, 16) || bad_stride(r.rb, padded(r.K)) || r.rb % 16))
      return set_error(TIERMM_EINVAL, "%s: int8 rows of %zu bytes (whole 16-byte units from %d up, 16-byte aligned)", who,
                       r.rb, padded(r.K));
  if (topk && (!sx || !expert_ids || !weights || !sgu || !sd)) return set_error(TIERMM_EINVAL, "%s: null table", who);
  if (misaligned(sx, 4) || misaligned(expert_ids, 4) || misaligned(weights, 4) || misaligned(sgu, 4) || misaligned(sd, 4))
    return set_error(TIERMM_EINVAL, "%s: misaligned table", who);
  if (misaligned(ws, 16)) return set_error(TIERMM_EINVAL, "%s: workspace not 16-byte aligned", who);
  const int P = T * topk, nt = (F + 15) / 16;
  void* w = nullptr;
  const int st = get_workspace(ws, ws_bytes, tiermm_moe_i8_layer_ws_bytes(T, topk, K, F), &w, who);
  if (st != TIERMM_OK) return st;
  float* h = (float*)w;
  float* y = (float*)((uint8_t*)w + align16((size_t)P * F * 4));
  uint32_t* top = (uint32_t*)((uint8_t*)y + align16((size_t)P * K * 4));
  const LayerArgs a = {(const uint8_t*)Xq, (const uint8_t*)Wgu, (const uint8_t*)Wd, sx, sgu, sd, weights, expert_ids, h, top, y,
                       (uint8_t*)out, rbx, rbg, rbd, ldo * es, T, topk, P, n_experts, K, F, padded(K) / 64, padded(F) / 64,
                       P < n_experts};
  hipStream_t s = (hipStream_t)stream;
  if (P) {
    const int slots = P < n_experts ? P : n_experts;
    moe_gate_up_kernel<<<dim3(nt, slots), 256, 0, s>>>(a);
    TM_LAUNCH_CHECK("tiermm_moe_i8_layer: gate and up");
    moe_down_kernel<<<dim3((K + 15) / 16, slots), 256, 0, s>>>(a);
    TM_LAUNCH_CHECK("tiermm_moe_i8_layer: down");
  }
  with_rows(otype, [&](auto yt) {
    moe_layer_sum_kernel<decltype(yt)::value><<<dim3(T, (K + 1023) / 1024), 256, 0, s>>>(a);
  });
  TM_LAUNCH_CHECK("tiermm_moe_i8_layer: sum");
  return TIERMM_OK;
}

}  // extern "C"
