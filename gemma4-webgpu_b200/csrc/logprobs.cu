// q4k_token_logprobs: log probabilities of given tokens, the entropy and the
// top alternatives of rows of logits, in one pass.  The reference takes 256
// raw candidates to the host and samples there (src/engine.ts:1792-1837); it
// has no log probabilities.
//
// Mathematics, in base 2 (y = x log2 e, x the softcapped logit): with a
// running maximum m,  s = sum 2^(y - m),  w = sum 2^(y - m) (y - m):
//   lse = ln 2 (m + log2 s),  entropy = ln 2 (log2 s - w / s).
// The softcap is monotone, so alternatives are chosen by the raw logits.
//
// A CTA takes a row, or a part of one when there are few rows, in tiles held
// in registers.  Each thread keeps its own (m, s, w).  Alternatives: the
// k-th largest of the threads' tile maxima bounds the k-th largest logit from
// below, so after the first tile only a few more than k elements pass the
// bound; they go to a list in shared memory that is cut back to k (by each
// entry's rank) when it has grown, which raises the bound.  A tile whose
// passing elements overflow the list (many equal logits) is searched k times
// instead.  The order is a 64-bit key, value then inverted index, so ties go
// to the lowest index and no two keys are equal: the result does not depend
// on the order of arrival.
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_cache.cuh"
#include "q4k_device.cuh"

namespace q4k {
namespace {

constexpr uint32_t kLpThreads = 256;
constexpr uint32_t kLpVecs = 4;      // 16-byte loads a thread and tile
constexpr uint32_t kLpTop = 32;      // most alternatives
constexpr uint32_t kLpList = 1024;   // list entries (kLpTop - 1 parts of kLpTop keys fit)
constexpr uint32_t kLpPrune = 64;    // entries at which the list is cut back
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct LpPart {  // what a part of a row leaves for the merge
  float m, s, w;
  uint32_t n;
  unsigned long long key[kLpTop];
};

struct LpArgs {
  const void* logits;
  uint64_t stride;
  uint32_t rows, V, splits, top;
  float cap;
  const int32_t* tokens;
  float* logprob;
  float* entropy;
  float* top_logprob;
  int32_t* top_token;
  LpPart* parts;       // [rows][splits]
  uint32_t* counters;  // [rows]
  uint32_t* status;
};

__device__ __forceinline__ float lp_ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

// Order of the values as whole numbers; NaN below everything, -0 = +0.
__device__ __forceinline__ uint32_t ord_of(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float of_ord(uint32_t o) {
  if (o == 0u) return __int_as_float(0x7fc00000);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ unsigned long long key_of(float x, uint32_t idx) {
  return ((unsigned long long)ord_of(x) << 32) | (0xffffffffu - idx);
}

// cap tanh(x / cap) = cap - 2 cap / (2^(2 log2(e) x / cap) + 1).
__device__ __forceinline__ float capped(float x, float cap) {
  if (cap <= 0.0f) return x;
  return cap - __fdividef(2.0f * cap, lp_ex2(x * (2.0f * kLog2e / cap)) + 1.0f);
}

struct Stats {
  float m, s, w;  // m = -inf: nothing yet
};
__device__ __forceinline__ void rebase(Stats& a, float m) {  // to a larger reference
  if (a.m == m) return;
  if (a.m != neg_inf()) {
    const float d = a.m - m, f = lp_ex2(d);
    // a.s == 0: nothing but -inf so far
    a.w = f * (a.w + a.s * max_nan(d, -252.0f));
    a.s *= f;
  }
  a.m = m;
}
__device__ __forceinline__ Stats merge(Stats a, Stats b) {
  const float m = fmaxf(a.m, b.m);
  rebase(a, m);
  rebase(b, m);
  return Stats{m, a.s + b.s, a.w + b.w};
}

// The list's entries by rank: the `k` largest first, in order.  All threads.
__device__ __forceinline__ uint32_t prune(unsigned long long* list, uint32_t n, uint32_t k) {
  __syncthreads();
  unsigned long long mine[kLpList / kLpThreads];
  uint32_t rank[kLpList / kLpThreads];
#pragma unroll
  for (uint32_t i = 0; i < kLpList / kLpThreads; ++i) {
    const uint32_t at = threadIdx.x + i * kLpThreads;
    mine[i] = at < n ? list[at] : 0ull;
    rank[i] = 0;
    if (at < n)
      for (uint32_t j = 0; j < n; ++j) rank[i] += list[j] > mine[i];
  }
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < kLpList / kLpThreads; ++i)
    if (mine[i] != 0ull && rank[i] < k) list[rank[i]] = mine[i];
  __syncthreads();
  return min(n, k);
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) logprobs_kernel(const LpArgs a) {
  constexpr uint32_t kVE = 16 / sizeof(T);  // elements of a vector
  constexpr uint32_t kN = kLpVecs * kVE;    // elements a thread and tile
  __shared__ unsigned long long s_list[kLpList];
  __shared__ unsigned long long s_key[kLpThreads / 32];
  __shared__ Stats s_stats[kLpThreads / 32];
  __shared__ uint32_t s_n, s_last;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const uint32_t row = blockIdx.x / a.splits, part = blockIdx.x % a.splits;
  const T* const x = static_cast<const T*>(a.logits) + (uint64_t)row * a.stride;
  // vectors of 16 aligned bytes; the first and last may hold elements of no row
  const uint32_t mis = (uint32_t)(((uintptr_t)x & 15u) / sizeof(T));
  const uint32_t n_vec = (a.V + mis + kVE - 1) / kVE, per = (n_vec + a.splits - 1) / a.splits;
  const uint32_t v_lo = min(part * per, n_vec), v_hi = min(v_lo + per, n_vec);
  const uint32_t k = a.top;

  Stats st{neg_inf(), 0.0f, 0.0f};
  uint32_t n_list = 0;      // entries of the list (the same in every thread)
  float bound = neg_inf();  // an element enters the list if above it
  bool first = true, equal = true;  // equal: also one equal to the bound
  if (tid == 0) s_n = 0;
  __syncthreads();

  for (uint32_t v0 = v_lo; v0 < v_hi; v0 += kLpThreads * kLpVecs, first = false) {
    float e[kN];
    uint32_t ok = 0;  // bit i: element i is one of the row's
    uint4 raw[kLpVecs];
#pragma unroll
    for (uint32_t i = 0; i < kLpVecs; ++i) {
      const uint32_t v = v0 + i * kLpThreads + tid;
      const bool in = v < v_hi && v * kVE >= mis && (v + 1) * kVE - mis <= a.V;
      if (in) {
        raw[i] = ldg_nc_v4(x + (int64_t)(v * kVE) - mis);
        ok |= ((1u << kVE) - 1u) << (i * kVE);
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < kLpVecs; ++i) {
      const uint32_t v = v0 + i * kLpThreads + tid;
      if (ok >> (i * kVE) & 1u) {
        const T* p = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
        for (uint32_t j = 0; j < kVE; ++j) e[i * kVE + j] = Elem<T>::to(p[j]);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < kVE; ++j) {
          const int64_t at = (int64_t)(v * kVE + j) - mis;
          e[i * kVE + j] = neg_inf();
          if (v < v_hi && at >= 0 && at < (int64_t)a.V) {
            e[i * kVE + j] = Elem<T>::to(x[at]);
            ok |= 1u << (i * kVE + j);
          }
        }
      }
    }
    float mx = e[0];
#pragma unroll
    for (uint32_t j = 1; j < kN; ++j) mx = fmaxf(mx, e[j]);

    // statistics
    {
      const float top = capped(mx, a.cap) * kLog2e;
      if (top > st.m) rebase(st, top);
      const float ref = st.m == neg_inf() ? 0.0f : st.m;
#pragma unroll
      for (uint32_t j = 0; j < kN; ++j) {
        const float d = max_nan(fmaf(capped(e[j], a.cap), kLog2e, -ref), -252.0f);  // 2^-252 is 0: -inf adds nothing
        const float p = lp_ex2(d);
        st.s += p;
        st.w = fmaf(p, d, st.w);
      }
    }
    if (k == 0) continue;

    // alternatives
    if (first) {
      const uint32_t mine = ok ? ord_of(mx) : 0u;
      uint32_t t = 0;  // the largest prefix that k threads' maxima reach
      for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
        if (__syncthreads_count(mine >= (t | bit)) >= (int)k) t |= bit;
      bound = t ? of_ord(t) : neg_inf();
      if (!(bound == bound)) bound = neg_inf();  // a prefix within NaN's codes
    }
    const bool mine = equal ? mx >= bound : mx > bound;
    if (mine) {
#pragma unroll
      for (uint32_t j = 0; j < kN; ++j) {
        if ((equal ? e[j] >= bound : e[j] > bound) && (ok >> j & 1u)) {
          const uint32_t at = atomicAdd(&s_n, 1u);
          const uint32_t v = v0 + (j / kVE) * kLpThreads + tid;
          if (at < kLpList) s_list[at] = key_of(e[j], v * kVE + j % kVE - mis);
        }
      }
    }
    if (!__syncthreads_or(mine) && !first) continue;
    uint32_t n = s_n;
    // the first tile owes k entries (or all that it has, were they NaN)
    const bool owe = first && n < k;
    if (n > kLpList || owe) {
      // search the tile itself: the largest key below the last, k times
      unsigned long long below = ~0ull;
      n = n_list;
      for (uint32_t r = 0; r < k; ++r) {
        unsigned long long best = 0;
#pragma unroll
        for (uint32_t j = 0; j < kN; ++j) {
          const uint32_t v = v0 + (j / kVE) * kLpThreads + tid;
          const unsigned long long key = key_of(e[j], v * kVE + j % kVE - mis);
          if ((ok >> j & 1u) && key < below && key > best) best = key;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
          best = other > best ? other : best;
        }
        __syncthreads();
        if (lane == 0) s_key[warp] = best;
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kLpThreads / 32; ++i) best = s_key[i] > best ? s_key[i] : best;
        if (best == 0) break;
        if (tid == 0) s_list[n] = best;
        ++n;
        below = best;
      }
    }
    if (first || n > kLpPrune) {
      n = prune(s_list, n, k);
      // later elements have higher indices: one equal to the k-th loses
      if (n == k) bound = of_ord((uint32_t)(s_list[k - 1] >> 32));
      equal = n < k || !(bound == bound);  // a NaN among the k yields to any number
      if (equal) bound = neg_inf();
    }
    n_list = n;
    __syncthreads();
    if (tid == 0) s_n = n;
    __syncthreads();
  }
  if (k && n_list > 0) n_list = prune(s_list, n_list, k);

  // the CTA's statistics, in thread 0's order of warps
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stats other;
    other.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    other.w = __shfl_xor_sync(0xffffffffu, st.w, o);
    st = merge(st, other);
  }
  if (lane == 0) s_stats[warp] = st;
  __syncthreads();
  st = s_stats[0];
#pragma unroll
  for (uint32_t i = 1; i < kLpThreads / 32; ++i) st = merge(st, s_stats[i]);

  if (a.splits > 1) {
    LpPart* const ps = a.parts + (uint64_t)row * a.splits;
    if (tid == 0) {
      ps[part].m = st.m;
      ps[part].s = st.s;
      ps[part].w = st.w;
      ps[part].n = n_list;
    }
    if (tid < k) ps[part].key[tid] = tid < n_list ? s_list[tid] : 0ull;
    __syncthreads();
    if (tid == 0) {
      __threadfence();
      s_last = atomicAdd(&a.counters[row], 1u) == a.splits - 1;
      if (s_last) a.counters[row] = 0;
      s_n = 0;
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    // parts in their order: thread i holds part i's statistics and largest key
    st = Stats{neg_inf(), 0.0f, 0.0f};
    for (uint32_t i = lane; i < a.splits; i += 32)
      st = merge(st, Stats{__ldcg(&ps[i].m), __ldcg(&ps[i].s), __ldcg(&ps[i].w)});
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Stats other;
      other.m = __shfl_xor_sync(0xffffffffu, st.m, o);
      other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
      other.w = __shfl_xor_sync(0xffffffffu, st.w, o);
      st = merge(st, other);
    }
    if (k) {
      // the k-th largest of the parts' first keys bounds the k-th largest key
      const unsigned long long head = tid < a.splits ? __ldcg(&ps[tid].key[0]) : 0ull;
      if (tid < a.splits) s_list[tid] = head;
      if (tid == 0) s_key[0] = 0;
      __syncthreads();
      if (tid < a.splits && a.splits >= k) {
        uint32_t rank = 0;
        for (uint32_t j = 0; j < a.splits; ++j) rank += s_list[j] > head;
        if (rank == k - 1) s_key[0] = head;
      }
      __syncthreads();
      const unsigned long long t = s_key[0];
      __syncthreads();
      for (uint32_t i = tid; i < a.splits * k; i += kLpThreads) {
        const unsigned long long key = __ldcg(&ps[i / k].key[i % k]);
        if (key != 0 && key >= t) s_list[atomicAdd(&s_n, 1u)] = key;
      }
      __syncthreads();
      n_list = prune(s_list, s_n, k);
    }
  }

  const float log_s = log2f(st.s);
  const bool empty = st.s == 0.0f;  // nothing above -inf
  const float lse = kLn2 * (st.m + log_s);
  if (tid == 0) {
    a.entropy[row] = empty ? 0.0f : kLn2 * (log_s - st.w / st.s);
    const int32_t tok = a.tokens[row];
    float lp = __int_as_float(0x7fc00000);
    if (tok >= 0 && (uint32_t)tok < a.V)
      lp = empty ? neg_inf() : capped(Elem<T>::to(x[tok]), a.cap) - lse;
    else if (tok >= 0)
      atomicOr(a.status, kStatusToken);
    a.logprob[row] = lp;
  }
  if (tid < k) {
    const unsigned long long key = s_list[tid];
    const uint64_t at = (uint64_t)row * k + tid;
    a.top_token[at] = (int32_t)(0xffffffffu - (uint32_t)key);
    a.top_logprob[at] = empty ? neg_inf() : capped(of_ord((uint32_t)(key >> 32)), a.cap) - lse;
  }
}

}  // namespace
}  // namespace q4k

using namespace q4k;

extern "C" int q4k_token_logprobs(q4k_ctx* ctx, uint32_t dtype, const void* logits, uint64_t stride, uint32_t rows,
                                  uint32_t V, float cap, const int32_t* tokens, uint32_t top, float* logprob,
                                  float* entropy, float* top_logprob, int32_t* top_token, void* stream) {
  if (!ctx) return Q4K_ERR_INVALID_ARG;
  if (dtype > Q4K_BF16) return ctx_fail(ctx, Q4K_ERR_INVALID_ARG, "q4k_token_logprobs: unknown dtype %u", dtype);
  if (rows == 0) {
    ctx->err[0] = 0;
    return Q4K_OK;
  }
  if (!logits || !tokens || !logprob || !entropy || (top && (!top_logprob || !top_token)))
    return ctx_fail(ctx, Q4K_ERR_INVALID_ARG, "q4k_token_logprobs: null pointer");
  if (V == 0 || V >= (1u << 30) || rows >= (1u << 24))
    return ctx_fail(ctx, Q4K_ERR_INVALID_ARG, "q4k_token_logprobs: V=%u or rows=%u out of range", V, rows);
  if (top > kLpTop || top > V)
    return ctx_fail(ctx, Q4K_ERR_INVALID_ARG, "q4k_token_logprobs: top=%u above %u or V=%u", top, kLpTop, V);
  if (stride < V) return ctx_fail(ctx, Q4K_ERR_INVALID_ARG, "q4k_token_logprobs: stride below V=%u", V);
  if (!(cap == cap)) return ctx_fail(ctx, Q4K_ERR_INVALID_ARG, "q4k_token_logprobs: cap is NaN");
  if ((uintptr_t)logits % dtype_bytes(dtype))
    return ctx_fail(ctx, Q4K_ERR_INVALID_ARG, "q4k_token_logprobs: logits not aligned to their type");
  LpArgs a{};
  a.logits = logits;
  a.stride = stride;
  a.rows = rows;
  a.V = V;
  a.top = top;
  a.cap = cap > 0.0f ? cap : 0.0f;
  a.tokens = tokens;
  a.logprob = logprob;
  a.entropy = entropy;
  a.top_logprob = top_logprob;
  a.top_token = top_token;
  a.parts = reinterpret_cast<LpPart*>(ctx->xfrag);
  a.counters = ctx->split_counters;
  a.status = ctx->select.status;
  // parts of a row: enough CTAs for every SM to hold several, no part below a tile
  const uint32_t tile = kLpThreads * kLpVecs * 16 / (uint32_t)dtype_bytes(dtype);
  const uint32_t want = (4 * (uint32_t)ctx->sm_count + rows - 1) / rows, most = (V + tile - 1) / tile;
  a.splits = want < most ? want : most;
  a.splits = a.splits > 64 ? 64 : a.splits;
  if (rows > kSplitCounters || (uint64_t)rows * a.splits * sizeof(LpPart) > ctx->xfrag_cap) a.splits = 1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == Q4K_F32)
    logprobs_kernel<float><<<rows * a.splits, kLpThreads, 0, st>>>(a);
  else if (dtype == Q4K_F16)
    logprobs_kernel<__half><<<rows * a.splits, kLpThreads, 0, st>>>(a);
  else
    logprobs_kernel<__nv_bfloat16><<<rows * a.splits, kLpThreads, 0, st>>>(a);
  return ctx_cuda(ctx, cudaGetLastError(), "q4k_token_logprobs launch");
}
