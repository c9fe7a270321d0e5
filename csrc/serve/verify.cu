// Verification of drafted tokens against the target model, from given random
// numbers.  Per sequence b with K drafted tokens x_i, target logits t [K + 1, V],
// draft logits d [K, V] (or none: the draft is certain of its tokens) and
// temperature T:
//   p_i = softmax(t_i / T),  q_i = softmax(d_i / T)  (or one at x_i)
//   x_i is accepted iff  u_i q_i(x_i) < p_i(x_i);  n = accepted before the first reject
//   next = argmax_j r_j / noise_j   (an exponential race: a draw from r)
//     r = max(p_n - q_n, 0) after a reject (p_n where that is all zero), p_n
//     after all lens[b] drafts were accepted
//   T = 0: x_i is accepted iff x_i = argmax t_i, next = argmax t_n (lowest index)
// Outputs: the accepted tokens, the next one, then -1; n; and log p of each
// emitted token (0 for T = 0).
//
// One cluster of CTAs per sequence, each CTA a slice of the vocabulary: it reads
// its slice of every row once, keeping the running maximum and sum of the
// softmax (per thread, then per CTA), the cluster exchanges the (max, sum) pairs
// through distributed shared memory, every CTA decides n alike, and the race
// over row n reads that one row again (from L2) with the noise, which is
// prefetched into L2 at the start.  One launch, no workspace.
//
// Bound by memory: 2 K + 1 rows of V logits and one row of noise per sequence.
#include <torch/extension.h>

#include "../common/host.h"
#include "../common/sm100.cuh"
#include "checks.h"

namespace hb {
namespace {

constexpr int VTHREADS = 512;
constexpr int VWARPS = VTHREADS / 32;
constexpr int VMAXROWS = 65;   // 2 K + 1 with K <= 32
constexpr float LOG2E_F = 1.4426950408889634f;
constexpr int NOIDX = 0x7fffffff;

struct VerifyParams {
  const void *target, *draft;         // [B, K + 1, V], [B, K, V] or null
  const long long* tokens;            // [B, K]
  const float *uniform, *noise, *temperature;   // [B, K], [B, V], [B] or null (temp)
  const int* lens;                    // [B] or null
  long long* out;                     // [B, K + 1]
  long long* accepted;                // [B]
  float* logp;                        // [B, K + 1]
  float temp;
  int B, K, V;
  int* status;
};

HB_DEVICE float vexp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One logit as fp32 with NaN read as minus infinity.
HB_DEVICE float as_logit(float x) { return x != x ? -INFINITY : x; }
HB_DEVICE float logit_at(const float* p, long long i) { return as_logit(p[i]); }
HB_DEVICE float logit_at(const __nv_bfloat16* p, long long i) { return as_logit(__bfloat162float(p[i])); }

// Elements per 16-byte load.
template <typename T>
struct Vec { static constexpr int N = 16 / sizeof(T); };
HB_DEVICE void unpack(uint4 u, float (&f)[4], const float*) {
  f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
}
HB_DEVICE void unpack(uint4 u, float (&f)[8], const __nv_bfloat16*) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// Running softmax statistics: m the maximum, s = sum e^{(l - m) / T}.
struct Stat {
  float m, s;
};
// e^{(a - b) / T} with c = log2(e) / T; equal arguments give 1 (infinities too).
HB_DEVICE float ratio(float a, float b, float c) { return a == b ? 1.f : vexp2((a - b) * c); }
HB_DEVICE Stat merge(Stat x, Stat y, float c) {
  const float m = fmaxf(x.m, y.m);
  if (m == -INFINITY) return {m, 0.f};
  return {m, x.s * ratio(x.m, m, c) + y.s * ratio(y.m, m, c)};
}
// softmax value of a logit from its row's statistics (0 for an empty row)
HB_DEVICE float prob(float x, Stat f, float inv) {
  return f.s > 0.f ? (x == f.m ? 1.f : expf((x - f.m) * inv)) / f.s : 0.f;
}
struct Best {   // greatest value, lowest index among equals
  float v;
  int i;
};
HB_DEVICE Best better(Best x, Best y) { return (y.v > x.v || (y.v == x.v && y.i < x.i)) ? y : x; }
HB_DEVICE Best warp_best(Best x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    x = better(x, Best{__shfl_xor_sync(0xffffffffu, x.v, o), __shfl_xor_sync(0xffffffffu, x.i, o)});
  return x;
}

// Calls vec(first index, values) for whole aligned 16-byte groups of row[c0, c1)
// and one(index, value) for the ragged ends.
template <typename T, int UNROLL, typename FV, typename F1>
HB_DEVICE void for_slice(const T* row, int c0, int c1, FV vec, F1 one) {
  constexpr int N = Vec<T>::N;
  const int tid = threadIdx.x, len = c1 - c0;
  if (len <= 0) return;
  const T* p = row + c0;
  const int mis = (int)((reinterpret_cast<uintptr_t>(p) / sizeof(T)) % N);
  const int head = min(len, mis ? N - mis : 0);
  const int nv = (len - head) / N, tail0 = head + nv * N;
  if (tid < head) one(c0 + tid, logit_at(p, tid));
  const uint4* pv = reinterpret_cast<const uint4*>(p + head);
  int i = tid;
  for (; i + (UNROLL - 1) * VTHREADS < nv; i += UNROLL * VTHREADS) {
    uint4 u[UNROLL];
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) u[j] = __ldg(pv + i + j * VTHREADS);
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      float f[N];
      unpack(u[j], f, p);
      vec(c0 + head + (i + j * VTHREADS) * N, f);
    }
  }
  for (; i < nv; i += VTHREADS) {
    float f[N];
    unpack(__ldg(pv + i), f, p);
    vec(c0 + head + i * N, f);
  }
  if (tid < len - tail0) one(c0 + tail0 + tid, logit_at(p, tail0 + tid));
}

HB_DEVICE float dsmem_f32(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(addr, rank)));
  return v;
}

template <typename T>
__global__ void __launch_bounds__(VTHREADS) verify_kernel(const VerifyParams p, const int cs) {
  constexpr int N = Vec<T>::N;
  __shared__ Stat part[VMAXROWS][VWARPS];   // per warp; then [.][0] is the CTA's
  __shared__ Best bpart[VMAXROWS][VWARPS];
  __shared__ Best rpart[2][VWARPS];         // of the race
  __shared__ Stat full[VMAXROWS];           // of the whole rows
  __shared__ int first[VMAXROWS];           // greedy: index of the row's maximum
  __shared__ float fin[4];                  // race results of this CTA: (score, index) twice
  __shared__ int s_n;

  const int b = blockIdx.x / cs, rank = blockIdx.x % cs;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int V = p.V, K = p.K;
  const int per = ((V + cs - 1) / cs + 63) / 64 * 64;
  const int c0 = min(V, rank * per), c1 = min(V, c0 + per);
  const T* tg = reinterpret_cast<const T*>(p.target) + (long long)b * (K + 1) * V;
  const T* dr = p.draft ? reinterpret_cast<const T*>(p.draft) + (long long)b * K * V : nullptr;
  const float* nz = p.noise + (long long)b * V;

  float temp = p.temperature ? p.temperature[b] : p.temp;
  const bool greedy = !(temp > 0.f);
  const float inv = greedy ? 1.f : 1.f / temp;
  const float cexp = inv * LOG2E_F;
  int L = K;
  if (p.lens) {
    const int x = p.lens[b];
    L = min(max(x, 0), K);
    if (x != L && tid == 0) set_error(p.status, kErrBounds);
  }
  const int nt = L + 1, rows = greedy || !dr ? nt : nt + L;   // row r < nt: target r, else draft r - nt

  if (!greedy)   // the race reads this slice of the noise at the end: bring it to L2 now
    for (int i = c0 + tid * 32; i < c1; i += VTHREADS * 32)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(nz + i));

  for (int r = 0; r < rows; ++r) {
    const T* row = r < nt ? tg + (long long)r * V : dr + (long long)(r - nt) * V;
    if (greedy) {
      Best best{-INFINITY, NOIDX};
      auto one = [&](int i, float x) {
        if (x > best.v || (x == best.v && x > -INFINITY && i < best.i)) best = {x, i};
      };
      for_slice<T, 4>(row, c0, c1,
                      [&](int i, const float(&f)[N]) {
#pragma unroll
                        for (int j = 0; j < N; ++j) one(i + j, f[j]);
                      },
                      one);
      best = warp_best(best);
      if (lane == 0) bpart[r][warp] = best;
    } else {
      Stat st{-INFINITY, 0.f};
      auto one = [&](int, float x) { st = merge(st, Stat{x, x > -INFINITY ? 1.f : 0.f}, cexp); };
      for_slice<T, 4>(row, c0, c1,
                      [&](int, const float(&f)[N]) {
                        float m = fmaxf(f[0], f[1]);   // fmaxf drops NaN
#pragma unroll
                        for (int j = 2; j < N; ++j) m = fmaxf(m, f[j]);
                        if (m > st.m) {
                          st.s *= vexp2((st.m - m) * cexp);   // 0 from the first maximum
                          st.m = m;
                        }
                        if (st.m > -INFINITY) {
#pragma unroll
                          for (int j = 0; j < N; ++j) {
                            const float e = f[j] == st.m ? 1.f : vexp2((f[j] - st.m) * cexp);
                            st.s += f[j] == f[j] ? e : 0.f;
                          }
                        }
                      },
                      one);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        st = merge(st, Stat{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o)}, cexp);
      if (lane == 0) part[r][warp] = st;
    }
  }
  __syncthreads();
  for (int r = warp; r < rows; r += VWARPS) {
    if (greedy) {
      Best x = lane < VWARPS ? bpart[r][lane] : Best{-INFINITY, NOIDX};
      x = warp_best(x);
      __syncwarp();
      if (lane == 0) bpart[r][0] = x;
    } else {
      Stat x = lane < VWARPS ? part[r][lane] : Stat{-INFINITY, 0.f};
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        x = merge(x, Stat{__shfl_xor_sync(0xffffffffu, x.m, o), __shfl_xor_sync(0xffffffffu, x.s, o)}, cexp);
      __syncwarp();
      if (lane == 0) part[r][0] = x;
    }
  }
  __syncwarp();
  cluster_sync_all();
  for (int r = tid; r < rows; r += VTHREADS) {   // every CTA merges all slices in the same order
    if (greedy) {
      Best x{-INFINITY, NOIDX};
      for (int c = 0; c < cs; ++c) {
        const uint32_t a = smem_u32(&bpart[r][0]);
        x = better(x, Best{dsmem_f32(a, c), __float_as_int(dsmem_f32(a + 4, c))});
      }
      first[r] = x.i;
    } else {
      Stat x{-INFINITY, 0.f};
      for (int c = 0; c < cs; ++c) {
        const uint32_t a = smem_u32(&part[r][0]);
        x = merge(x, Stat{dsmem_f32(a, c), dsmem_f32(a + 4, c)}, cexp);
      }
      full[r] = x;
    }
  }
  __syncthreads();
  if (warp == 0) {   // acceptance, 32 drafted positions at a time (K <= 32)
    bool ok = false;
    if (lane < L) {
      const long long x = p.tokens[(long long)b * K + lane];
      if (index_ok(x, V, p.status)) {
        if (greedy) {
          ok = (int)x == first[lane];
        } else {
          const float pt = prob(logit_at(tg, (long long)lane * V + x), full[lane], inv);
          float qt = 1.f;
          if (dr) qt = prob(logit_at(dr, (long long)lane * V + x), full[nt + lane], inv);
          ok = p.uniform[(long long)b * K + lane] * qt < pt;
        }
      }
    }
    const unsigned rej = ~__ballot_sync(0xffffffffu, ok);
    if (lane == 0) s_n = min(L, rej ? __ffs(rej) - 1 : 32);
  }
  __syncthreads();
  const int n = s_n;

  // the race over row n: residual scores and, in case every residual is 0, p's own
  Best res{0.f, NOIDX}, own{0.f, NOIDX};
  if (!greedy) {
    const Stat ft = full[n];
    const bool minus = n < L;
    const Stat fd = minus && dr ? full[nt + n] : Stat{0.f, 0.f};
    const long long taken = minus && !dr ? p.tokens[(long long)b * K + n] : -1;
    const T* trow = tg + (long long)n * V;
    const T* drow = minus && dr ? dr + (long long)n * V : nullptr;
    if (ft.s > 0.f)
      for (int i = c0 + tid; i < c1; i += VTHREADS) {
        const float pj = prob(logit_at(trow, i), ft, inv), e = nz[i];
        float r = pj;
        if (drow) r = fmaxf(pj - prob(logit_at(drow, i), fd, inv), 0.f);
        if (i == taken) r = 0.f;
        const float sr = r / e, so = pj / e;
        if (sr > res.v) res = {sr, i};
        if (so > own.v) own = {so, i};
      }
  }
  res = warp_best(res), own = warp_best(own);
  if (lane == 0) rpart[0][warp] = res, rpart[1][warp] = own;
  __syncthreads();
  if (warp == 0) {
    Best x = warp_best(lane < VWARPS ? rpart[0][lane] : Best{0.f, NOIDX});
    Best y = warp_best(lane < VWARPS ? rpart[1][lane] : Best{0.f, NOIDX});
    if (lane == 0) {
      fin[0] = x.v, fin[1] = __int_as_float(x.i);
      fin[2] = y.v, fin[3] = __int_as_float(y.i);
    }
  }
  __syncwarp();
  cluster_sync_all();
  if (rank == 0 && warp == 0) {
    int next;
    if (greedy) {
      next = first[n];
    } else {
      Best x{0.f, NOIDX}, y{0.f, NOIDX};
      for (int c = 0; c < cs; ++c) {
        const uint32_t a = smem_u32(fin);
        x = better(x, Best{dsmem_f32(a, c), __float_as_int(dsmem_f32(a + 4, c))});
        y = better(y, Best{dsmem_f32(a + 8, c), __float_as_int(dsmem_f32(a + 12, c))});
      }
      next = x.v > 0.f ? x.i : y.i;
    }
    for (int i = lane; i <= K; i += 32) {
      long long tok = -1;
      if (i < n) tok = p.tokens[(long long)b * K + i];
      else if (i == n) tok = next < V ? next : -1;
      float lp = 0.f;
      if (tok >= 0 && !greedy) {
        const Stat f = full[i];
        const float x = logit_at(tg, (long long)i * V + tok);
        lp = (x == f.m ? 0.f : (x - f.m) * inv) - logf(f.s);
      }
      p.out[(long long)b * (K + 1) + i] = tok;
      p.logp[(long long)b * (K + 1) + i] = lp;
    }
    if (lane == 0) p.accepted[b] = n;
  }
  __syncwarp();
  cluster_sync_all();   // the peers' shared memory is read until here
}

template <typename T>
void launch_verify(const VerifyParams& p) {
  // Enough CTAs for two waves' worth of SMs, slices of at least 1024 logits.
  int cs = 8;
  while (cs > 1 && ((long long)p.B * cs > 4 * num_sms() || p.V / cs < 1024)) cs /= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)p.B * cs);
  cfg.blockDim = dim3(VTHREADS);
  cfg.stream = cur_stream();
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = cs, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  HB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_kernel<T>, p, cs));
}

}  // namespace

// target [B, K + 1, V], draft [B, K, V] or none -> tokens [B, K + 1], accepted
// [B], log probabilities [B, K + 1].
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> verify_draft(torch::Tensor target, torch::Tensor tokens,
                                                                     torch::Tensor uniform, torch::Tensor noise,
                                                                     OptTensor draft, OptTensor lens,
                                                                     OptTensor temperature, double temp) {
  const auto dev = target.device();
  const c10::cuda::CUDAGuard guard(dev);
  need(target.dim() == 3 && target.size(1) >= 1 && target.size(2) >= 1, "verify_draft: target logits [B, K + 1, V]");
  need(target.scalar_type() == at::kFloat || target.scalar_type() == at::kBFloat16, "verify_draft: fp32 or bf16 logits");
  const int64_t B = target.size(0), K = target.size(1) - 1, V = target.size(2);
  need(K <= 32, "verify_draft: at most 32 drafted tokens");
  need(V < (1ll << 30), "verify_draft: at most 2^30 logits a row");
  const auto is = [&](const torch::Tensor& t, int64_t n, at::ScalarType ty) {
    return t.dim() == 2 && t.size(0) == B && t.size(1) == n && t.scalar_type() == ty && t.device() == dev;
  };
  need(is(tokens, K, at::kLong), "verify_draft: drafted tokens [B, K] int64");
  need(is(uniform, K, at::kFloat), "verify_draft: uniform [B, K] fp32");
  need(is(noise, V, at::kFloat), "verify_draft: noise [B, V] fp32");
  if (draft)
    need(draft->dim() == 3 && draft->size(0) == B && draft->size(1) == K && draft->size(2) == V &&
             draft->scalar_type() == target.scalar_type() && draft->device() == dev,
         "verify_draft: draft logits [B, K, V] of the target's type");
  if (lens) lens = whole(*lens, B, dev, "verify_draft: draft_lens, B whole numbers on the logits' device");
  if (temperature) {
    need(temperature->dim() == 1 && temperature->size(0) == B && temperature->scalar_type() == at::kFloat &&
             temperature->device() == dev,
         "verify_draft: temperature [B] fp32, or a number");
    temperature = temperature->contiguous();
  }
  need(!wants_grad(target) && !(draft && wants_grad(*draft)), "verify_draft has no backward: call it under torch.no_grad()");
  const auto opt = target.options();
  torch::Tensor out = torch::empty({B, K + 1}, opt.dtype(at::kLong)), accepted = torch::empty({B}, opt.dtype(at::kLong)),
                logp = torch::empty({B, K + 1}, opt.dtype(at::kFloat));
  if (B == 0) return {out, accepted, logp};
  target = target.contiguous(), tokens = tokens.contiguous(), uniform = uniform.contiguous(), noise = noise.contiguous();
  if (draft) draft = draft->contiguous();
  VerifyParams p{};
  p.B = (int)B, p.K = (int)K, p.V = (int)V;
  p.target = target.data_ptr();
  p.draft = draft ? draft->data_ptr() : nullptr;
  p.tokens = (const long long*)tokens.data_ptr<int64_t>();
  p.uniform = uniform.data_ptr<float>(), p.noise = noise.data_ptr<float>();
  p.temperature = temperature ? temperature->data_ptr<float>() : nullptr;
  p.lens = lens ? lens->data_ptr<int>() : nullptr;
  p.out = (long long*)out.data_ptr<int64_t>(), p.accepted = (long long*)accepted.data_ptr<int64_t>();
  p.logp = logp.data_ptr<float>();
  p.temp = (float)temp;
  p.status = status_ptr();
  if (target.scalar_type() == at::kFloat) launch_verify<float>(p);
  else launch_verify<__nv_bfloat16>(p);
  return {out, accepted, logp};
}

}  // namespace hb
