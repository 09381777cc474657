// moe_layer.hip -- a routed layer of a few tokens over int8 experts: gate and up, the gate's
// activation, down, and the weighted sum of a token's experts, in two kernels for few pairs and four
// for more.  No reference function (the reference refuses MoE models, arch.py:158-159).
//
//   g, u = int8 products of x with an expert's gate and up rows (tm_i8.h: exact sums, fp32 scales)
//   h = fp32(silu(g) u), in 64 bits, rounded once
//   hq = codes of h's row, scale max|h| / 127, as tiermm_i8_quant makes them
//   out[t] = sum_j weights[t][j] * (int8 product of hq with the down rows), in j order in fp32
//
// 64 bits for the gate: h is then the same fp32 number whatever exp does in its last bits, and its
// codes with it.
#include "tm_i8.h"
#include "tm_tiles.h"

namespace tiermm {
namespace {

constexpr int kTokens = TIERMM_MOE_LAYER_TOKENS, kTopk = TIERMM_MOE_LAYER_TOPK, kPairs = kTokens * kTopk;

struct LayerArgs {
  const uint8_t *X, *Wg, *Wd;        // codes: T rows, E * 2F rows (gate, then up), E * K rows
  const float *sx, *sg, *sd, *weights;
  const int32_t* ids;
  float* h;                          // [P][F]
  uint32_t* top;                     // [P][tiles of F]: largest |h|, as bits
  uint8_t* hq;                       // [P][padded F] codes of h
  float* sh;                         // [P]
  float* y;                          // [P][K]
  uint32_t* arrived;                 // [tiles of K] workgroups of moe_down_few_kernel that are done, cleared by the gate's
  uint8_t* out;
  size_t rbx, rbg, rbd, ldo;         // bytes
  int T, topk, P, E, K, F, nk, nf;   // nk, nf: 128-byte steps of x's and h's rows
  int by_pair;                       // slots are pairs (fewer than experts): the first of an expert's acts
};

// The pairs of this workgroup's expert, in order, into list; returns their number (0: nothing to do).
// An id outside [0, E) is a dropped pair.
__device__ __forceinline__ int find_pairs(const LayerArgs& a, int slot, int& e, uint16_t* list) {
  const int lane = threadIdx.x & 63;
  int id = a.ids[min(lane, a.P - 1)];  // on its way with the slot's own
  e = a.by_pair ? a.ids[slot] : slot;
  asm volatile("" : "+v"(id));
  if ((uint32_t)e >= (uint32_t)a.E) return 0;
  int n = 0;
  for (int p0 = 0; p0 < a.P; p0 += 64) {
    const int p = p0 + lane;
    if (p0) id = a.ids[min(p, a.P - 1)];
    const uint64_t hit = __ballot(p < a.P && id == e);
    if (a.by_pair && hit && n == 0 && p0 + __ffsll((unsigned long long)hit) - 1 < slot) return 0;
    // (every wave writes the same list)
    if (hit >> lane & 1) list[n + __popcll(hit & ((1ull << lane) - 1))] = (uint16_t)p;
    n += __popcll(hit);
  }
  return n;
}

constexpr int kFew = 8;             // pairs of an expert that moe_down_few_kernel takes at a time
constexpr int kFewCols = 32;        // its columns of out a workgroup
constexpr int kTile = 16;           // columns of h whose largest magnitude is kept

// An expert's tokens, BM at a time, times COLS rows of its weight.  DOWN false: half of them the gate's and the same of
// up, x the tokens' codes, h out.  DOWN true: x the codes of h, the pairs' fp32 products out.
//
// Bound by the weights' bytes: a ring of S stages of 128 bytes of every row (x's, then W's) keeps S - 1 on their way by
// global_load_lds, whole lines of eight rows a load; the four waves share the columns and the two 64-byte steps, one
// barrier a stage.  An expert of more than BM pairs goes through its weights again, out of the caches.
//
// Four workgroups a CU, each with a small ring, hide one another's start (its pairs, then its first weights) and
// end.  8 of 64 experts of 2048 x 1408, gate and up: 8 tokens 40.5 us (6.0 TB/s), 64 tokens 69 (5.3); the whole
// call 71 and 113.  Rings of 80 KB, two workgroups a CU: 94 and 164.
template <int BM, int COLS, int S, bool DOWN>
__global__ __launch_bounds__(256) void moe_experts_kernel(const LayerArgs a) {
  constexpr int MB = BM / 16, HALF = COLS / 2, NB = HALF / 16, ROWS = BM + COLS;
  constexpr int STAGE = ROWS * kStep, INST = STAGE / 1024 / 4, LDO = COLS + 4;
  static_assert(INST * 4 * 1024 == STAGE && 2 * BM * LDO * 4 <= S * STAGE, "whole loads a wave, sums in LDS");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ uint16_t list[kPairs];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int e;
  if (!DOWN && blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = tid; i < (a.K + kFewCols - 1) / kFewCols; i += 256) a.arrived[i] = 0;
  const int n = find_pairs(a, blockIdx.y, e, list);
  if (n == 0) return;
  const int n0 = blockIdx.x * (DOWN ? COLS : HALF), N = DOWN ? a.K : a.F, nk = DOWN ? a.nf : a.nk;
  const size_t rbw = DOWN ? a.rbd : a.rbg, rbx = DOWN ? (size_t)a.nf * kStep : a.rbx;
  const uint8_t* W = DOWN ? a.Wd + (size_t)e * a.K * rbw : a.Wg + (size_t)e * 2 * a.F * rbw;
  auto w_row = [&](int r) { return DOWN ? min(n0 + r, N - 1) : (r < HALF ? 0 : N) + min(n0 + r % HALF, N - 1); };
  const uint32_t lds0 = lds_addr(lds);
  const int wn = wave & 1, wk = wave >> 1, fr = lane & 15, fg = lane >> 4, turn = (fr >> 1) & 7;
  __syncthreads();
  for (int base = 0; base < n; base += BM) {
    // load u of this wave: eight rows of a stage
    const uint8_t* src[INST];
#pragma unroll
    for (int u = 0; u < INST; ++u) {
      const int r = 8 * (wave + 4 * u) + (lane >> 3);
      const int p = list[min(base + r, n - 1)];  // (of a row of W: not used)
      src[u] = (r < BM ? (DOWN ? a.hq : a.X) + (size_t)(DOWN ? p : p / a.topk) * rbx : W + (size_t)w_row(r - BM) * rbw) +
               ((lane & 7) ^ ((r >> 1) & 7)) * 16;
    }
    int put = 0;
    auto issue = [&](int st) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < INST; ++u) {
        const uint8_t* from = src[u] + (size_t)st * kStep;
        const uint32_t to = lds0 + put * STAGE + (wave + 4 * u) * 1024;
        if (8 * (wave + 4 * u) >= BM && n <= BM) dma16_nt(from, to);
        else dma16(from, to);
      }
      put = put + 1 == S ? 0 : put + 1;
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
      if (i < nk) issue(i);
    i32x4 acc[NB][MB] = {};
    int get = 0;
    for (int st = 0; st < nk; ++st) {
      const int after = nk - 1 - st;  // stages on their way behind this one
      if (after >= S - 2) vm_wait<(S - 2) * INST>();
      else wait_stages<S - 3, INST>(after);
      __syncthreads();  // stage st has landed for every wave, and the one before it is read
      if (st + S - 1 < nk) issue(st + S - 1);
      const uint8_t* s = lds + get * STAGE;
      get = get + 1 == S ? 0 : get + 1;
      const uint8_t* p = s + fr * kStep + ((4 * wk + fg) ^ turn) * 16;
      i32x4 xf[MB], wf[NB];
#pragma unroll
      for (int i = 0; i < MB; ++i) xf[i] = *(const i32x4*)(p + i * 16 * kStep);
#pragma unroll
      for (int j = 0; j < NB; ++j) wf[j] = *(const i32x4*)(p + (BM + wn * HALF + j * 16) * kStep);
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], xf[i], acc[j][i], 0, 0, 0);
    }
    __syncthreads();
    // a lane's sum is columns 4 * fg .. + 3 of row fr of each block
    int32_t* sums = (int32_t*)lds;
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < MB; ++i) *(i32x4*)(sums + (wk * BM + i * 16 + fr) * LDO + wn * HALF + j * 16 + 4 * fg) = acc[j][i];
    __syncthreads();
    if constexpr (DOWN) {
      for (int q = tid; q < BM * COLS; q += 256) {
        const int r = q / COLS, c = q % COLS;
        if (base + r >= n || n0 + c >= N) continue;
        const int p = list[base + r], sum = sums[r * LDO + c] + sums[(BM + r) * LDO + c];
        a.y[(size_t)p * a.K + n0 + c] = scaled(sum, a.sh[p], a.sd[(size_t)e * a.K + n0 + c], 0.f);
      }
    } else {
      for (int q = tid; q < BM * HALF; q += 256) {
        const int r = q / HALF, c = q % HALF, p = list[min(base + r, n - 1)];
        const bool live = base + r < n;
        uint32_t top = 0;
        if (live && n0 + c < N) {
          const int32_t* g = sums + r * LDO + c;
          const size_t ch = (size_t)e * 2 * N + n0 + c;
          const float sx = a.sx[p / a.topk];
          const double gate = scaled(g[0] + g[BM * LDO], sx, a.sg[ch], 0.f);
          const double up = scaled(g[HALF] + g[BM * LDO + HALF], sx, a.sg[ch + N], 0.f);
          const float h = (float)(gate / (1. + exp(-gate)) * up);
          a.h[(size_t)p * N + n0 + c] = h;
          top = __float_as_uint(h) & 0x7fffffffu;
        }
#pragma unroll
        for (int o = kTile / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, kTile));
        if (c % kTile == 0 && live && n0 + c < N) a.top[(size_t)p * ((N + kTile - 1) / kTile) + (n0 + c) / kTile] = top;
      }
    }
    __syncthreads();
  }
}

// Down for few pairs: 32 rows of an expert's weight times the codes of its rows of h, kFew at a time, which each
// workgroup makes for itself while its first weights are on the way; then the last of the workgroups that share the
// columns adds the tokens' experts.  That spares two launches and repeats the codes in every workgroup: 8 of 64
// experts of 2048 x 1408, the whole call with it and with moe_codes_kernel, moe_experts_kernel and
// moe_layer_sum_kernel: 1 token 21.4 and 23.7 us, 2 tokens 33.6 and 35.4, 4 tokens 52.2 and 53.1, 8 tokens 74.3 and
// 70.5; 2 of 8 experts of 4096 x 2816 1 token 22.8 and 26.1, 8 tokens 61.7 and 59.2, 16 tokens 75 and 64.
constexpr int kFewPairs = 32, kFewCodes = 24 * 1024;  // pairs, and bytes of codes in LDS (three workgroups a CU)
bool takes_few(int P, int F) { return P <= kFewPairs && kFew * padded(F) <= kFewCodes; }

template <int KS, int S, int YT>
__global__ __launch_bounds__(256) void moe_down_few_kernel(const LayerArgs a) {
  using Y = Rows<YT>;
  constexpr int COLS = kFewCols, SUB = COLS * kStep, STAGE = KS * SUB, INST = STAGE / 1024 / 4, LDO = COLS + 4;
  static_assert(INST * 4 * 1024 == STAGE && 2 * 16 * LDO * 4 <= S * STAGE, "whole loads a wave, sums in LDS");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // ring, then codes [kFew][padded F]
  __shared__ uint16_t list[kPairs];
  __shared__ float scale[kFew];
  __shared__ uint32_t turn_of;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * COLS, Fp = a.nf * kStep, nk = a.nf, ns = (nk + KS - 1) / KS;
  int e;
  const int n = find_pairs(a, blockIdx.y, e, list);
  uint8_t* codes = lds + S * STAGE;
  const uint32_t lds0 = lds_addr(lds);
  const int wn = wave & 1, wk = wave >> 1, fr = lane & 15, fg = lane >> 4, turn = (fr >> 1) & 7;
  __syncthreads();
  for (int base = 0; base < n; base += kFew) {
    const uint8_t* src[INST];
#pragma unroll
    for (int u = 0; u < INST; ++u) {
      const int r = (8 * (wave + 4 * u) + (lane >> 3)) % COLS;
      src[u] = a.Wd + ((size_t)e * a.K + min(n0 + r, a.K - 1)) * a.rbd + ((lane & 7) ^ ((r >> 1) & 7)) * 16;
    }
    int put = 0;
    auto issue = [&](int st) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < INST; ++u) {
        const size_t k = (size_t)min(KS * st + 8 * (wave + 4 * u) / COLS, nk - 1) * kStep;  // (past the end: not multiplied)
        dma16_nt(src[u] + k, lds0 + put * STAGE + (wave + 4 * u) * 1024);
      }
      put = put + 1 == S ? 0 : put + 1;
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
      if (i < ns) issue(i);
    // codes of the rows: 16-byte chunk c of row r at chunk c ^ r of its 128 bytes
    const int rows = min(kFew, n - base), nt = (a.F + kTile - 1) / kTile;
    for (int r = 0; r < rows; ++r) {
      const int p = list[base + r];
      const uint8_t* h = (const uint8_t*)(a.h + (size_t)p * a.F);
      auto load = [&](int f) { return f < a.F ? Rows<QT_F32>::get(h, f, a.F) : u32x4{0u, 0u, 0u, 0u}; };
      const u32x4 h0 = load(tid * 4), h1 = load(tid * 4 + 1024);  // on their way while the scale is found
      uint32_t top = 0;
      for (int i = lane; i < nt; i += 64) top = max(top, a.top[(size_t)p * nt + i]);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
      const RowScale rs = row_scale_of(top);
      if (tid == 0) scale[r] = rs.sc;
      auto put = [&](int f, u32x4 u) {
        float v[4];
        Rows<QT_F32>::widen(u, v);
        *(uint32_t*)(codes + r * Fp + (f ^ (r << 4))) = codes4(v, rs);
      };
      if (tid * 4 < Fp) put(tid * 4, h0);
      if (tid * 4 + 1024 < Fp) put(tid * 4 + 1024, h1);
      for (int f = tid * 4 + 2048; f < Fp; f += 1024) put(f, load(f));
    }
    i32x4 acc = {0, 0, 0, 0};
    const int xr = min(fr, rows - 1);
    int get = 0;
    for (int st = 0; st < ns; ++st) {
      const int after = ns - 1 - st;  // stages on their way behind this one
      if (after >= S - 2) vm_wait<(S - 2) * INST>();
      else wait_stages<S - 3, INST>(after);
      __syncthreads();  // stage st has landed for every wave (and the codes are there), and the one before it is read
      if (st + S - 1 < ns) issue(st + S - 1);
      const uint8_t* s = lds + get * STAGE + (wn * 16 + fr) * kStep;
      get = get + 1 == S ? 0 : get + 1;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int step = wk * KS + k, sub = step >> 1, c = 4 * (step & 1) + fg;
        if (KS * st + sub >= nk) break;
        const i32x4 wf = *(const i32x4*)(s + sub * SUB + (c ^ turn) * 16);
        const i32x4 xf = *(const i32x4*)(codes + xr * Fp + (KS * st + sub) * kStep + (c ^ xr) * 16);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, xf, acc, 0, 0, 0);
      }
    }
    __syncthreads();
    int32_t* sums = (int32_t*)lds;  // a lane's sum is columns 4 * fg .. + 3 of row fr
    *(i32x4*)(sums + (wk * 16 + fr) * LDO + wn * 16 + 4 * fg) = acc;
    __syncthreads();
    const int r = tid / COLS, c = tid % COLS;
    static_assert(kFew * COLS == 256, "a sum a thread");
    if (r < rows && n0 + c < a.K) {
      const float v = scaled(sums[r * LDO + c] + sums[(16 + r) * LDO + c], scale[r], a.sd[(size_t)e * a.K + n0 + c], 0.f);
      __hip_atomic_store(a.y + (size_t)list[base + r] * a.K + n0 + c, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
  }
  // The workgroups of these columns count themselves, and the last one finds every product written: products and counts are
  // stored and loaded at the scope of the device, past the L2 of one XCD, every wave has waited for its stores in front of
  // its workgroup's count, and the last one's loads are issued behind its own.  (A release and an acquire fence instead,
  // which write back and invalidate the caches: 8 tokens 251 us.)
  vm_wait<0>();
  __syncthreads();
  if (tid == 0) turn_of = __hip_atomic_fetch_add(a.arrived + blockIdx.x, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (turn_of != gridDim.y - 1) return;
  const int cols = min(COLS, a.K - n0);
  for (int t = tid / COLS; t < a.T; t += 256 / COLS) {
    const int c = tid % COLS;
    if (c >= cols) continue;
    float v = 0.f;
    for (int j0 = 0; j0 < a.topk; j0 += 8) {
      float w[8], y[8];
      bool live[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int p = t * a.topk + min(j0 + j, a.topk - 1);
        live[j] = j0 + j < a.topk && (uint32_t)a.ids[p] < (uint32_t)a.E;
        w[j] = live[j] ? a.weights[p] : 0.f;
        y[j] = live[j] ? __hip_atomic_load(a.y + (size_t)p * a.K + n0 + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v = live[j] ? fmaf(w[j], y[j], v) : v;  // (adding 0 would lose a zero's sign)
    }
    const float o[4] = {v, 0.f, 0.f, 0.f};
    Y::put4(a.out + (size_t)t * a.ldo + (size_t)(n0 + c) * Y::ES, o, 1);
  }
}

// Codes and scale of a pair's row of h.
__global__ __launch_bounds__(256) void moe_codes_kernel(const LayerArgs a) {
  __shared__ uint32_t red[4];
  const int p = blockIdx.x, tid = threadIdx.x, nt = (a.F + kTile - 1) / kTile, Fp = a.nf * kStep;
  if ((uint32_t)a.ids[p] >= (uint32_t)a.E) return;
  uint32_t top = 0;
  for (int i = tid; i < nt; i += 256) top = max(top, a.top[(size_t)p * nt + i]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if ((tid & 63) == 0) red[tid >> 6] = top;
  __syncthreads();
  const RowScale rs = row_scale_of(max(max(red[0], red[1]), max(red[2], red[3])));
  const uint8_t* h = (const uint8_t*)(a.h + (size_t)p * a.F);
  for (int f = (blockIdx.y * 256 + tid) * 4; f < Fp; f += gridDim.y * 1024) {
    float v[4];
    Rows<QT_F32>::widen(f < a.F ? Rows<QT_F32>::get(h, f, a.F) : u32x4{0u, 0u, 0u, 0u}, v);
    *(uint32_t*)(a.hq + (size_t)p * Fp + f) = codes4(v, rs);
  }
  if (blockIdx.y == 0 && tid == 0) a.sh[p] = rs.sc;
}

template <int BM, int COLS, int S, bool DOWN>
int launch_experts(const LayerArgs& a, int slots, hipStream_t s, const char* who) {
  constexpr int LDS = S * (BM + COLS) * kStep;
  static std::atomic<uint64_t> done{0};
  const int st = lds_attr_once(done, (const void*)moe_experts_kernel<BM, COLS, S, DOWN>, LDS, who);
  if (st != TIERMM_OK) return st;
  const int n = DOWN ? COLS : COLS / 2;
  moe_experts_kernel<BM, COLS, S, DOWN><<<dim3(((DOWN ? a.K : a.F) + n - 1) / n, slots), 256, LDS, s>>>(a);
  TM_LAUNCH_CHECK(who);
  return TIERMM_OK;
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

template <int KS, int S, int YT>
int launch_few(const LayerArgs& a, int slots, hipStream_t s, const char* who) {
  constexpr int RING = S * KS * kFewCols * kStep;
  static_assert(RING + kFewCodes + kPairs * 2 + 64 <= 64 * 1024, "LDS that a launch has without asking");
  const int lds = RING + kFew * a.nf * kStep;  // (takes_few)
  moe_down_few_kernel<KS, S, YT><<<dim3((a.K + kFewCols - 1) / kFewCols, slots), 256, lds, s>>>(a);
  TM_LAUNCH_CHECK(who);
  return TIERMM_OK;
}

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

}  // namespace
}  // namespace tiermm

using namespace tiermm;

extern "C" {

size_t tiermm_moe_i8_layer_ws_bytes(int T, int topk, int K, int F) {
  if (T < 1 || topk < 1 || K < 1 || F < 1 || T > kTokens || topk > kTopk || K > kMaxK || F > kMaxK) return 0;
  const size_t P = (size_t)T * topk;
  return align16(P * F * 4) + align16(P * K * 4) + align16(P * ((F + kTile - 1) / kTile) * 4) + P * padded(F) + align16(P * 4) +
         align16((size_t)(K + kFewCols - 1) / kFewCols * 4);
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
  const int P = T * topk;
  void* w = nullptr;
  int st = get_workspace(ws, ws_bytes, tiermm_moe_i8_layer_ws_bytes(T, topk, K, F), &w, who);
  if (st != TIERMM_OK) return st;
  uint8_t* at = (uint8_t*)w;
  auto part = [&](size_t bytes) {
    uint8_t* p = at;
    at += align16(bytes);
    return p;
  };
  float* h = (float*)part((size_t)P * F * 4);
  float* y = (float*)part((size_t)P * K * 4);
  uint32_t* top = (uint32_t*)part((size_t)P * ((F + kTile - 1) / kTile) * 4);
  uint8_t* hq = part((size_t)P * padded(F));
  float* sh = (float*)part((size_t)P * 4);
  uint32_t* arrived = (uint32_t*)part((size_t)(K + kFewCols - 1) / kFewCols * 4);
  const LayerArgs a = {(const uint8_t*)Xq, (const uint8_t*)Wgu, (const uint8_t*)Wd, sx, sgu, sd, weights, expert_ids, h, top, hq, sh,
                       y, arrived, (uint8_t*)out, rbx, rbg, rbd, ldo * es, T, topk, P, n_experts, K, F, padded(K) / kStep, padded(F) / kStep,
                       P < n_experts};
  hipStream_t s = (hipStream_t)stream;
  if (P) {
    const int slots = P < n_experts ? P : n_experts;
    // Few pairs take tiles of half the columns, so that every CU has some.  us with half and whole tiles: 64 experts
    // of 1408, top 8 (K 2048) 1 token 21.4 / 22.6, 2 tokens 33.6 / 31.5, 4 tokens 51.7 / 52.5, 8 tokens 73.8 / 71.4,
    // 64 tokens 129 / 114; 8 of 2816, top 2 (K 4096) 1 token 22.8 / 26.7, 4 tokens 42.0 / 43.4, 8 tokens 61.5 / 60.2;
    // 128 of 768, top 4 (K 2048) 4 tokens 22.5 / 23.4, 8 tokens 37.3 / 34.5.
    const bool small = P <= 16;
    st = small ? launch_experts<32, 32, 4, false>(a, slots, s, who) : launch_experts<32, 64, 3, false>(a, slots, s, who);
    if (st != TIERMM_OK) return st;
    if (takes_few(P, F)) {
      with_rows(otype, [&](auto yt) { st = launch_few<2, 3, decltype(yt)::value>(a, slots, s, who); });
      return st;
    }
    moe_codes_kernel<<<dim3(P, (padded(F) + 4095) / 4096), 256, 0, s>>>(a);
    TM_LAUNCH_CHECK(who);
    st = small ? launch_experts<32, 32, 4, true>(a, slots, s, who) : launch_experts<32, 64, 3, true>(a, slots, s, who);
    if (st != TIERMM_OK) return st;
  }
  with_rows(otype, [&](auto yt) {
    moe_layer_sum_kernel<decltype(yt)::value><<<dim3(T, (K + 1023) / 1024), 256, 0, s>>>(a);
  });
  TM_LAUNCH_CHECK("tiermm_moe_i8_layer: sum");
  return TIERMM_OK;
}

}  // extern "C"
