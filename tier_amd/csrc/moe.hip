// moe.hip -- routed tokens on their way to the experts and back: the order of the
// (token, expert) pairs, the rows in that order, the weighted sum that brings them
// back, and the gradients of both.  No reference function (the reference refuses MoE
// models, arch.py:158-159).
//
// All are bound by memory: a row is read or written once, in 16-byte units, with the
// few indices of a token in scalar registers.  No atomics on results: every sum has one
// owner and one order, so results do not change between runs.  Measured on 4096 tokens,
// top 8 of 64, rows of 2048, between buffers that the caches do not hold (a large copy moves
// 5.1 TB/s): sort 53 us fp32 (5.7 TB/s), 27 us bf16; its gradient 54 and 27; the weighted sum's
// 27.5 in bf16 (5.5); that one's gradient 115 and 62 (4.7-4.9, the same bytes read as written).
// Eight tokens: 2.2 to 2.6 us replayed from a graph, 3.0 to 3.4 launched one by one.
#include "tm_rows.h"

namespace tiermm {
namespace {

// -------------------------------------------------------------------- plan
// Place of pair i (expert_ids[i], i = t * topk + j) in the order by (expert, i): the
// number of pairs of lower experts plus the number of earlier pairs of its own.
//
// One workgroup per expert (and one for the dropped pairs, as expert E) reads all ids:
// it counts those below and the earlier ones of its own, and writes its own places.
// That is E + 1 reads of P ids through L2, but one launch and no exchange between
// workgroups: 32768 pairs, 64 experts 7.6 us, where the two launches below take 8.3.  A tile
// is 4 ids a thread; NT tiles stay in registers (16 of them spilled: the limit of 8).
constexpr int kPlanMost = 8 * 4096;
typedef int32_t i32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

template <int THREADS, int NT>
__global__ __launch_bounds__(THREADS) void moe_plan_kernel(const int32_t* __restrict__ ids, int P, int E,
                                                                int32_t* __restrict__ offsets,
                                                                int32_t* __restrict__ places,
                                                                int32_t* __restrict__ sorted) {
  constexpr int NW = THREADS / 64, TILE = 4 * THREADS;
  __shared__ int own[NT * NW], less[NW];
  const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint64_t below = (1ull << lane) - 1;
  int first[NT];      // pairs of this expert before this thread's, within its wave and tile
  uint32_t mine = 0;  // bit 4t + i: id i of tile t's four is of this expert
  int lt = 0;
  i32x4_a4 id[NT];  // every load on its way before the first is used
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int i0 = t * TILE + 4 * tid;
    if ((t + 1) * TILE <= P) {
      id[t] = *(const i32x4_a4*)(ids + i0);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) id[t][i] = i0 + i < P ? ids[i0 + i] : -1;
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int i0 = t * TILE + 4 * tid;
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int v = id[t][i], key = (uint32_t)v < (uint32_t)E ? v : E;
      lt += key < e;
      m |= (uint32_t)(key == e && i0 + i < P) << i;
    }
    mine |= m << (4 * t);
    // prefix over the wave of counts 0..4, from the ballots of their three bits
    const int c = __popc(m);
    const uint64_t b0 = __ballot(c & 1), b1 = __ballot(c & 2), b2 = __ballot(c & 4);
    first[t] = __popcll(b0 & below) + 2 * __popcll(b1 & below) + 4 * __popcll(b2 & below);
    if (lane == 0) own[t * NW + wave] = __popcll(b0) + 2 * __popcll(b1) + 4 * __popcll(b2);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) lt += __shfl_xor(lt, o, 64);
  if (lane == 0) less[wave] = lt;
  __syncthreads();
  if (wave == 0) {  // own[] becomes the place of each (tile, wave)'s first pair
    int run = lane < NW ? less[lane] : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) run += __shfl_xor(run, o, 64);
    if (lane == 0) offsets[e] = run;
#pragma unroll
    for (int q = 0; q < NT * NW; q += 64) {
      const int n = q + lane < NT * NW ? own[q + lane] : 0;
      int s = n;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(s, o, 64);
        s += lane >= o ? up : 0;
      }
      if (q + lane < NT * NW) own[q + lane] = run + s - n;
      run += __shfl(s, 63, 64);
    }
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const uint32_t m = mine >> (4 * t);
    int at = own[t * NW + wave] + first[t];
    const int i0 = t * TILE + 4 * tid;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (m >> i & 1) {
        sorted[at] = e < E ? i0 + i : -1;
        places[i0 + i] = e < E ? at : -1;
        ++at;
      }
  }
}

// Longer batches: a histogram of each chunk of pairs, then one workgroup per chunk that adds
// the histograms before its own and places its pairs (524288 pairs, 256 experts: 26 us).
// Each workgroup reads every chunk's histogram, so long batches take longer chunks; the work still
// grows with the square of the chunks: 2^23 pairs, 1024 experts 1.08 ms, 64 experts' 524288 pairs 20 us.
constexpr int kChunkWaves = 4;
constexpr int plan_chunk(long long P) { return P <= 256 * 1024 ? 1024 : 4096; }

__global__ __launch_bounds__(64 * kChunkWaves) void moe_hist_kernel(const int32_t* __restrict__ ids, int P, int E,
                                                                    int chunk, int32_t* __restrict__ hist) {
  extern __shared__ int cnt[];
  for (int e = threadIdx.x; e <= E; e += 64 * kChunkWaves) cnt[e] = 0;
  __syncthreads();
  const int end = min(P, (int)(blockIdx.x + 1) * chunk);
  for (int i = blockIdx.x * chunk + threadIdx.x; i < end; i += 64 * kChunkWaves) {
    const int id = ids[i];
    atomicAdd(&cnt[(uint32_t)id < (uint32_t)E ? id : E], 1);  // whole numbers: any order
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += 64 * kChunkWaves) hist[(size_t)blockIdx.x * (E + 1) + e] = cnt[e];
}

// LDS: next[kChunkWaves][E + 1], the place of each wave's next pair of each expert, and total[E + 1].
__global__ __launch_bounds__(64 * kChunkWaves) void moe_place_kernel(const int32_t* __restrict__ ids, int P, int E,
                                                                     int chunk, int nb,
                                                                     const int32_t* __restrict__ hist,
                                                                     int32_t* __restrict__ offsets,
                                                                     int32_t* __restrict__ places,
                                                                     int32_t* __restrict__ sorted) {
  extern __shared__ int lds[];
  const int K = E + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
  int* next = lds;
  int* total = lds + kChunkWaves * K;
  for (int e = tid; e < K; e += 64 * kChunkWaves) {
    int all = 0, before = 0;
#pragma unroll 16
    for (int c = 0; c < nb; ++c) {
      const int n = hist[(size_t)c * K + e];
      all += n;
      before += c < b ? n : 0;
    }
    total[e] = all;
    next[e] = before;  // of wave 0 for now
#pragma unroll
    for (int w = 1; w < kChunkWaves; ++w) next[w * K + e] = 0;
  }
  __syncthreads();
  // counts of waves 0 .. kChunkWaves-2 into the next wave's start
  const int per = chunk / kChunkWaves, w0 = b * chunk + wave * per, w1 = min(P, w0 + per);
  if (wave + 1 < kChunkWaves)
    for (int i = w0 + lane; i < w1; i += 64) {
      const int id = ids[i];
      atomicAdd(&next[(wave + 1) * K + ((uint32_t)id < (uint32_t)E ? id : E)], 1);
    }
  __syncthreads();
  // starts of the experts: a prefix of total[], by the first wave
  if (wave == 0) {
    int run = 0;
    for (int e0 = 0; e0 < K; e0 += 64) {
      const int e = e0 + lane, n = e < K ? total[e] : 0;
      int s = n;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(s, o, 64);
        s += lane >= o ? up : 0;
      }
      if (e < K) {
        total[e] = run + s - n;
        if (b == 0) offsets[e] = run + s - n;  // offsets[E]: where the dropped pairs start
      }
      run += __shfl(s, 63, 64);
    }
  }
  __syncthreads();
  for (int e = tid; e < K; e += 64 * kChunkWaves) {
    int at = total[e];
#pragma unroll
    for (int w = 0; w < kChunkWaves; ++w) {
      at += next[w * K + e];
      next[w * K + e] = at;
    }
  }
  __syncthreads();
  // a wave places 64 pairs at a time: the lanes of the same expert are found from the
  // ballots of the key's bits, the last of them moves the expert's next place on
  const int kb = 32 - __clz(E);  // bits of the keys 0..E
  for (int i = w0; i < w1; i += 64) {
    const bool in = i + lane < w1;
    const int id = in ? ids[i + lane] : 0, key = (uint32_t)id < (uint32_t)E ? id : E;
    uint64_t same = __ballot(in);
    for (int k = 0; k < kb; ++k) {
      const uint64_t v = __ballot(key >> k & 1);
      same &= key >> k & 1 ? v : ~v;
    }
    if (in) {
      const int rank = __popcll(same & ((1ull << lane) - 1));
      const int at = next[wave * K + key] + rank;
      sorted[at] = key < E ? i + lane : -1;
      places[i + lane] = key < E ? at : -1;
      if (same >> lane == 1) next[wave * K + key] = at + 1;
    }
    // the next 64 read what the last lanes wrote: one wave's LDS operations stay in order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// -------------------------------------------------------------------- rows
struct RowArgs {
  const uint8_t* x;     // rows read
  uint8_t* y;           // rows written
  const int32_t* places;
  const int32_t* sorted;
  const float* w;
  size_t ldx, ldy;      // bytes
  int P, topk, cols;
};

// Xs[places[t][j]] = X[t]: a token's row is read once and written topk times, by the
// workgroups of blockIdx.x = t, 256 units each.  Those of token t also clear the rows
// t * topk .. + topk - 1 of Xs that hold no pair.
//
// NT: the copies go past the caches, where rows are whole 16-byte units: 59 -> 53 us in fp32 at
// 4096 tokens, top 8, 2048 columns, 30 -> 27 in bf16, between buffers that the caches do not
// hold; on rows of 2047 bf16, whose units straddle lines, 36 -> 39.  With a reader behind it (the
// int8 quantizer, which then finds the rows in memory), both together, through the caches -> past
// them, fp32: 8 tokens 5.1 -> 5.4 us, 128 7.7 -> 7.5, 512 16.2 -> 16.8, 4096 108 -> 119; bf16: 8
// 5.1 -> 5.3, 128 7.1 -> 7.2, 512 12.6 -> 12.4, 4096 68 -> 69.
template <int XT, bool NT>
__global__ __launch_bounds__(256) void moe_sort_kernel(const RowArgs a) {
  using R = Rows<XT>;
  const int t = blockIdx.x, c = (blockIdx.y * 256 + threadIdx.x) * R::EPU;
  if (c >= a.cols) return;
  const u32x4 u = R::get(a.x + (size_t)t * a.ldx, c, a.cols);
  for (int j0 = 0; j0 < a.topk; j0 += 8) {
    int p[8], pair[8];  // eight places' loads at a time, before the first store
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = t * a.topk + min(j0 + j, a.topk - 1);
      p[j] = a.places[i];
      pair[j] = a.sorted[i];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j0 + j >= a.topk) break;
      if ((uint32_t)p[j] < (uint32_t)a.P) {
        uint8_t* row = a.y + (size_t)p[j] * a.ldy;
        if constexpr (NT) R::set_nt(row, c, a.cols, u);
        else R::set(row, c, a.cols, u);
      }
      if (pair[j] < 0) R::set(a.y + (size_t)(t * a.topk + j0 + j) * a.ldy, c, a.cols, u32x4{0u, 0u, 0u, 0u});
    }
  }
}

// out[t] = sum_j w[t][j] Ys[places[t][j]], in j order in fp32 (WEIGHTED false: w = 1).
// Eight rows are in flight at a time.
//
// NT: rows of more bytes in all than the last-level cache keeps from one call to the next are
// read past it: 68 -> 54 us in fp32 at 4096 tokens, top 8, 2048 columns (256 MiB), 26.5 -> 24.6
// at 80 MiB, but 7.5 -> 7.7 at 32 and 12.2 -> 13.7 at 64; on rows of 1023 bf16 16 -> 20.
constexpr size_t kStreamBytes = 72 << 20;
template <int XT, bool WEIGHTED, bool NT>
__global__ __launch_bounds__(256) void moe_gather_sum_kernel(const RowArgs a) {
  using R = Rows<XT>;
  const int t = blockIdx.x, c = (blockIdx.y * 256 + threadIdx.x) * R::EPU;
  if (c >= a.cols) return;
  float acc[R::EPU];
#pragma unroll
  for (int i = 0; i < R::EPU; ++i) acc[i] = 0.f;
  for (int j0 = 0; j0 < a.topk; j0 += 8) {
    u32x4 u[8];
    int p[8];
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = t * a.topk + min(j0 + j, a.topk - 1);
      p[j] = j0 + j < a.topk ? a.places[i] : -1;
      w[j] = WEIGHTED ? a.w[i] : 1.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if ((uint32_t)p[j] < (uint32_t)a.P) u[j] = NT ? R::get_nt(a.x + (size_t)p[j] * a.ldx, c, a.cols)
                                                 : R::get(a.x + (size_t)p[j] * a.ldx, c, a.cols);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if ((uint32_t)p[j] >= (uint32_t)a.P) continue;
      float v[R::EPU];
      R::widen(u[j], v);
#pragma unroll
      for (int i = 0; i < R::EPU; ++i) acc[i] = WEIGHTED ? fmaf(w[j], v[i], acc[i]) : acc[i] + v[i];
    }
  }
  R::set(a.y + (size_t)t * a.ldy, c, a.cols, R::narrow(acc));
}

struct UnsortGradArgs {
  const uint8_t *dout, *ys;
  uint8_t* dys;
  const int32_t *places, *sorted;
  const float* w;
  float* dw;
  size_t ldo, ldy, ldd;  // bytes
  int P, topk, cols;
};

// dYs[p] = w dout[t] and dw[t][j] = <dout[t], Ys[p]> of pair (t, j) at place p, by one
// workgroup: dout comes from L2 for all but a token's first pair.  (A workgroup a token, dout
// read once: 138 against 119 us in fp32 at 4096 tokens, 10.3 against 4.2 at 128.)  The rows
// of dYs are stored past the caches: 118 -> 115 us, and 89 -> 68 on rows of 2047 bf16; with a reader
// behind it 8 tokens 5.1 -> 5.4 us, 512 26.8 -> 27.7, 4096 172 -> 172 (fp32).
template <int XT>
__global__ __launch_bounds__(256) void moe_unsort_grad_kernel(const UnsortGradArgs a) {
  using R = Rows<XT>;
  __shared__ float part[4];
  const int i = blockIdx.x, t = i / a.topk, p = a.places[i], tid = threadIdx.x;
  const bool live = (uint32_t)p < (uint32_t)a.P;
  const float w = live ? a.w[i] : 0.f;
  float s = 0.f;
  if (live)
    for (int c = tid * R::EPU; c < a.cols; c += 256 * R::EPU) {
      float d[R::EPU], y[R::EPU];
      R::widen(R::get(a.dout + (size_t)t * a.ldo, c, a.cols), d);
      R::widen(R::get(a.ys + (size_t)p * a.ldy, c, a.cols), y);
#pragma unroll
      for (int k = 0; k < R::EPU; ++k) {
        s = fmaf(d[k], y[k], s);
        d[k] *= w;
      }
      R::set_nt(a.dys + (size_t)p * a.ldd, c, a.cols, R::narrow(d));
    }
  if (a.sorted[i] < 0)
    for (int c = tid * R::EPU; c < a.cols; c += 256 * R::EPU)
      R::set(a.dys + (size_t)i * a.ldd, c, a.cols, u32x4{0u, 0u, 0u, 0u});
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((tid & 63) == 0) part[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) a.dw[i] = (part[0] + part[1]) + (part[2] + part[3]);
}

// Checks shared by the row entry points; *es = bytes of an element.
int check_rows(const char* who, int xtype, int T, int topk, int cols, int* es) {
  *es = row_elem_bytes(xtype);
  if (!*es) return set_error(TIERMM_UNSUPPORTED, "%s: rows of type %d", who, xtype);
  if (T < 0 || topk < 0 || cols < 0) return set_error(TIERMM_EINVAL, "%s: negative size", who);
  if (T > TIERMM_MOE_MAX_PAIRS || (long long)T * topk > TIERMM_MOE_MAX_PAIRS)
    return set_error(TIERMM_UNSUPPORTED, "%s: %d x %d pairs", who, T, topk);
  return TIERMM_OK;
}
bool misaligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) != 0; }
bool stream_rows(const void* rows, const RowArgs& a) {
  return !misaligned(rows, 16) && a.ldx % 16 == 0 && (size_t)a.P * a.ldx >= kStreamBytes;
}

}  // namespace
}  // namespace tiermm

using namespace tiermm;

extern "C" {

size_t tiermm_moe_plan_ws_bytes(int T, int topk, int n_experts) {
  if (T < 0 || topk < 0 || n_experts < 1) return 0;
  const long long P = (long long)T * topk;
  if (P <= kPlanMost) return 0;
  return (size_t)((P + plan_chunk(P) - 1) / plan_chunk(P)) * (n_experts + 1) * sizeof(int32_t);
}

int tiermm_moe_plan(const int32_t* expert_ids, int T, int topk, int n_experts, int32_t* expert_offsets,
                    int32_t* token_pairs, int32_t* sorted_pairs, void* ws, size_t ws_bytes, tiermm_stream_t stream) {
  const char* who = "tiermm_moe_plan";
  if (T < 0 || topk < 0 || n_experts < 1) return set_error(TIERMM_EINVAL, "%s: bad size", who);
  if (n_experts > TIERMM_MOE_MAX_EXPERTS)
    return set_error(TIERMM_UNSUPPORTED, "%s: %d experts, at most %d", who, n_experts, TIERMM_MOE_MAX_EXPERTS);
  const long long pairs = (long long)T * topk;
  if (pairs > TIERMM_MOE_MAX_PAIRS) return set_error(TIERMM_UNSUPPORTED, "%s: %d x %d pairs", who, T, topk);
  const int P = (int)pairs, E = n_experts;
  if (!expert_offsets || (P && (!expert_ids || !token_pairs || !sorted_pairs)))
    return set_error(TIERMM_EINVAL, "%s: null buffer", who);
  if (misaligned(expert_ids, 4) || misaligned(expert_offsets, 4) || misaligned(token_pairs, 4) ||
      misaligned(sorted_pairs, 4))
    return set_error(TIERMM_EINVAL, "%s: misaligned table", who);
  hipStream_t s = (hipStream_t)stream;
  const size_t need = tiermm_moe_plan_ws_bytes(T, topk, E);
  if (need) {
    void* hist = nullptr;
    const int st = get_workspace(ws, ws_bytes, need, &hist, who);
    if (st != TIERMM_OK) return st;
    const int chunk = plan_chunk(P), nb = (P + chunk - 1) / chunk;
    moe_hist_kernel<<<nb, 64 * kChunkWaves, (E + 1) * sizeof(int), s>>>(expert_ids, P, E, chunk, (int32_t*)hist);
    TM_LAUNCH_CHECK("tiermm_moe_plan: histogram");
    moe_place_kernel<<<nb, 64 * kChunkWaves, (kChunkWaves + 1) * (E + 1) * sizeof(int), s>>>(
        expert_ids, P, E, chunk, nb, (const int32_t*)hist, expert_offsets, token_pairs, sorted_pairs);
    TM_LAUNCH_CHECK("tiermm_moe_plan: places");
    return TIERMM_OK;
  }
#define PLAN(THREADS, NT) moe_plan_kernel<THREADS, NT><<<E + 1, THREADS, 0, s>>>(expert_ids, P, E, expert_offsets, token_pairs, sorted_pairs)
  if (P <= 1024) PLAN(256, 1);
  else if (P <= 4096) PLAN(1024, 1);
  else if (P <= 2 * 4096) PLAN(1024, 2);
  else if (P <= 4 * 4096) PLAN(1024, 4);
  else PLAN(1024, 8);
#undef PLAN
  TM_LAUNCH_CHECK("tiermm_moe_plan: launch");
  return TIERMM_OK;
}

int tiermm_moe_sort(const void* X, int xtype, size_t ldx, const int32_t* token_pairs, const int32_t* sorted_pairs,
                    void* X_sorted, size_t lds, int T, int topk, int K, tiermm_stream_t stream) {
  const char* who = "tiermm_moe_sort";
  int es;
  const int st = check_rows(who, xtype, T, topk, K, &es);
  if (st != TIERMM_OK) return st;
  if (bad_stride(ldx, K) || bad_stride(lds, K)) return set_error(TIERMM_EINVAL, "%s: row stride below %d or past 2^40", who, K);
  if (T == 0 || topk == 0 || K == 0) return TIERMM_OK;
  if (!X || !token_pairs || !sorted_pairs || !X_sorted) return set_error(TIERMM_EINVAL, "%s: null buffer", who);
  if (misaligned(X, es) || misaligned(X_sorted, es) || misaligned(token_pairs, 4) || misaligned(sorted_pairs, 4))
    return set_error(TIERMM_EINVAL, "%s: misaligned buffer", who);
  const RowArgs a = {(const uint8_t*)X, (uint8_t*)X_sorted, token_pairs, sorted_pairs, nullptr,
                     ldx * es, lds * es, T * topk, topk, K};
  const dim3 grid(T, (K * (size_t)es + 4095) / 4096);
  const bool whole = !misaligned(X_sorted, 16) && lds * es % 16 == 0;
  with_rows(xtype, [&](auto xt) {
    constexpr int XT = decltype(xt)::value;
    if (whole) moe_sort_kernel<XT, true><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    else moe_sort_kernel<XT, false><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  });
  TM_LAUNCH_CHECK("tiermm_moe_sort: launch");
  return TIERMM_OK;
}

int tiermm_moe_sort_grad(const void* dX_sorted, int xtype, size_t lds, const int32_t* token_pairs, void* dX, size_t ldx,
                         int T, int topk, int K, tiermm_stream_t stream) {
  const char* who = "tiermm_moe_sort_grad";
  int es;
  const int st = check_rows(who, xtype, T, topk, K, &es);
  if (st != TIERMM_OK) return st;
  if (bad_stride(ldx, K) || bad_stride(lds, K)) return set_error(TIERMM_EINVAL, "%s: row stride below %d or past 2^40", who, K);
  if (T == 0 || K == 0) return TIERMM_OK;
  if (!dX || (topk && (!dX_sorted || !token_pairs))) return set_error(TIERMM_EINVAL, "%s: null buffer", who);
  if (misaligned(dX_sorted, es) || misaligned(dX, es) || misaligned(token_pairs, 4))
    return set_error(TIERMM_EINVAL, "%s: misaligned buffer", who);
  const RowArgs a = {(const uint8_t*)dX_sorted, (uint8_t*)dX, token_pairs, nullptr, nullptr,
                     lds * es, ldx * es, T * topk, topk, K};
  const dim3 grid(T, (K * (size_t)es + 4095) / 4096);
  with_rows(xtype, [&](auto xt) {
    constexpr int XT = decltype(xt)::value;
    if (stream_rows(dX_sorted, a)) moe_gather_sum_kernel<XT, false, true><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    else moe_gather_sum_kernel<XT, false, false><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  });
  TM_LAUNCH_CHECK("tiermm_moe_sort_grad: launch");
  return TIERMM_OK;
}

int tiermm_moe_unsort(const void* Y_sorted, int ytype, size_t lds, const int32_t* token_pairs, const float* weights,
                      void* out, size_t ldo, int T, int topk, int N, tiermm_stream_t stream) {
  const char* who = "tiermm_moe_unsort";
  int es;
  const int st = check_rows(who, ytype, T, topk, N, &es);
  if (st != TIERMM_OK) return st;
  if (bad_stride(ldo, N) || bad_stride(lds, N)) return set_error(TIERMM_EINVAL, "%s: row stride below %d or past 2^40", who, N);
  if (T == 0 || N == 0) return TIERMM_OK;
  if (!out || (topk && (!Y_sorted || !token_pairs || !weights)))
    return set_error(TIERMM_EINVAL, "%s: null buffer", who);
  if (misaligned(Y_sorted, es) || misaligned(out, es) || misaligned(token_pairs, 4) || misaligned(weights, 4))
    return set_error(TIERMM_EINVAL, "%s: misaligned buffer", who);
  const RowArgs a = {(const uint8_t*)Y_sorted, (uint8_t*)out, token_pairs, nullptr, weights,
                     lds * es, ldo * es, T * topk, topk, N};
  const dim3 grid(T, (N * (size_t)es + 4095) / 4096);
  with_rows(ytype, [&](auto xt) {
    constexpr int XT = decltype(xt)::value;
    if (stream_rows(Y_sorted, a)) moe_gather_sum_kernel<XT, true, true><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    else moe_gather_sum_kernel<XT, true, false><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  });
  TM_LAUNCH_CHECK("tiermm_moe_unsort: launch");
  return TIERMM_OK;
}

int tiermm_moe_unsort_grad(const void* dout, int ytype, size_t ldo, const void* Y_sorted, size_t lds,
                           const int32_t* token_pairs, const int32_t* sorted_pairs, const float* weights,
                           void* dY_sorted, size_t ldd, float* dweights, int T, int topk, int N,
                           tiermm_stream_t stream) {
  const char* who = "tiermm_moe_unsort_grad";
  int es;
  const int st = check_rows(who, ytype, T, topk, N, &es);
  if (st != TIERMM_OK) return st;
  if (bad_stride(ldo, N) || bad_stride(lds, N) || bad_stride(ldd, N))
    return set_error(TIERMM_EINVAL, "%s: row stride below %d or past 2^40", who, N);
  if (T == 0 || topk == 0) return TIERMM_OK;
  if (!token_pairs || !sorted_pairs || !weights || !dweights || (N && (!dout || !Y_sorted || !dY_sorted)))
    return set_error(TIERMM_EINVAL, "%s: null buffer", who);
  if (misaligned(dout, es) || misaligned(Y_sorted, es) || misaligned(dY_sorted, es) || misaligned(token_pairs, 4) ||
      misaligned(sorted_pairs, 4) || misaligned(weights, 4) || misaligned(dweights, 4))
    return set_error(TIERMM_EINVAL, "%s: misaligned buffer", who);
  const UnsortGradArgs a = {(const uint8_t*)dout, (const uint8_t*)Y_sorted, (uint8_t*)dY_sorted, token_pairs,
                            sorted_pairs, weights, dweights, ldo * es, lds * es, ldd * es, T * topk, topk, N};
  with_rows(ytype, [&](auto xt) {
    moe_unsort_grad_kernel<decltype(xt)::value><<<T * topk, 256, 0, (hipStream_t)stream>>>(a);
  });
  TM_LAUNCH_CHECK("tiermm_moe_unsort_grad: launch");
  return TIERMM_OK;
}

}  // extern "C"
