// The gated delta rule token by token, with its state (model/kda.py:305-323):
//   S <- diag(e^g) S;   u = beta (v - beta S^T k);   S <- S + k u^T;   o = scale S^T q
// for tokens t < counts[b], per (sequence, head), S [K, V] fp32 (V = K).
//
// Every column of S evolves by itself, so a CTA owns VC columns of one (b, h)
// and the columns need no exchange.  A column's K rows lie in RG lanes of one
// warp, R rows each, in registers for the whole call: the state is read once and
// written once whatever the number of tokens.  Token rows (q, k, e^g, v, beta)
// are staged TC at a time in shared memory, the next TC already in registers.
//
// Bound: with one token the state traffic (8 K V bytes); with many tokens the
// dependent chain of a token (R multiply-adds, two or three shuffles, R more).
#include <torch/extension.h>

#include "../common/host.h"
#include "../common/sm100.cuh"
#include "checks.h"

namespace hb {
namespace {

struct Row3 {   // strides in elements of [B, S, H, (K)]
  long long b, s, h;
};
struct RecParams {
  const void *q, *k, *v;
  const float *g, *beta;
  Row3 qs, ks, vs, gs, bs;
  const float* s0;            // [B, H, K, K] with batch stride s0_b (0: shared), or null
  long long s0_b;
  float *s1, *o;              // contiguous
  const int* counts;
  int B, S, H;
  float scale;
  int* status;
};

template <typename T>
HB_DEVICE float to_f(T x);
template <>
HB_DEVICE float to_f(float x) { return x; }
template <>
HB_DEVICE float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

template <int CPT>
HB_DEVICE void ldc(const float* p, float (&x)[CPT]) {
  if constexpr (CPT == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else if constexpr (CPT == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    x[0] = v.x, x[1] = v.y;
  } else {
    x[0] = *p;
  }
}
template <int CPT>
HB_DEVICE void stc(float* p, const float (&x)[CPT]) {
  if constexpr (CPT == 4) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  else if constexpr (CPT == 2) *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
  else *p = x[0];
}

// K rows, RG lanes per column group of CPT columns, VC columns per CTA, TC
// staged tokens.
template <typename T, int K, int RG, int CPT, int VC, int TC>
__global__ void __launch_bounds__(VC / CPT * RG) kda_recurrent_kernel(const RecParams p) {
  constexpr int R = K / RG;
  constexpr int THREADS = VC / CPT * RG;
  constexpr int CL = 32 / RG;               // column groups per warp
  constexpr int SEG = R + 4;                // padded rows of one lane group: distinct banks per group
  constexpr int ROW = RG * SEG;
  constexpr int NE = (TC * K + THREADS - 1) / THREADS;   // staged q (k, g) elements per thread
  constexpr int NV = (TC * VC + THREADS - 1) / THREADS;
  __shared__ __align__(16) float sq[TC * ROW], sk[TC * ROW], sa[TC * ROW];
  __shared__ __align__(16) float sv[TC * VC];
  __shared__ float sb[TC];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rg = lane / CL;                               // row group
  const int c0 = (warp * CL + lane % CL) * CPT;           // first column within the CTA's slice
  constexpr int SLICES = K / VC;
  const int slice = blockIdx.x % SLICES;
  const long long bh = blockIdx.x / SLICES;
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const int col = slice * VC + c0;

  float st[R][CPT];
  const float* s0 = p.s0 ? p.s0 + b * p.s0_b + ((long long)h * K + rg * R) * K + col : nullptr;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (s0) ldc<CPT>(s0 + r * K, st[r]);
    else
#pragma unroll
      for (int c = 0; c < CPT; ++c) st[r][c] = 0.f;
  }

  int n = p.S;
  if (p.counts) {
    const int c = p.counts[b];
    n = min(max(c, 0), p.S);
    if (c != n && tid == 0) set_error(p.status, kErrBounds);
  }
  const T* q = reinterpret_cast<const T*>(p.q) + b * p.qs.b + h * p.qs.h;
  const T* k = reinterpret_cast<const T*>(p.k) + b * p.ks.b + h * p.ks.h;
  const T* v = reinterpret_cast<const T*>(p.v) + b * p.vs.b + h * p.vs.h + slice * VC;
  const float* g = p.g + b * p.gs.b + h * p.gs.h;
  const float* be = p.beta + b * p.bs.b + h * p.bs.h;
  float* o = p.o + ((long long)b * p.S * p.H + h) * K + slice * VC;

  float rq[NE], rk[NE], ra[NE], rv[NV], rb = 0.f;
  auto fetch = [&](int t0) {
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const int idx = e * THREADS + tid, t = t0 + idx / K, i = idx % K;
      const bool in = (TC * K % THREADS == 0 || idx < TC * K) && t < n;
      rq[e] = in ? to_f(q[t * p.qs.s + i]) : 0.f;
      rk[e] = in ? to_f(k[t * p.ks.s + i]) : 0.f;
      ra[e] = in ? g[t * p.gs.s + i] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < NV; ++e) {
      const int idx = e * THREADS + tid, t = t0 + idx / VC;
      rv[e] = (TC * VC % THREADS == 0 || idx < TC * VC) && t < n ? to_f(v[t * p.vs.s + idx % VC]) : 0.f;
    }
    rb = tid < TC && t0 + tid < n ? be[(t0 + tid) * p.bs.s] : 0.f;
  };
  auto stage = [&]() {
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const int idx = e * THREADS + tid;
      if (TC * K % THREADS == 0 || idx < TC * K) {
        const int t = idx / K, i = idx % K, at = t * ROW + i / R * SEG + i % R;
        sq[at] = rq[e] * p.scale;
        sk[at] = rk[e];
        sa[at] = expf(ra[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < NV; ++e) {
      const int idx = e * THREADS + tid;
      if (TC * VC % THREADS == 0 || idx < TC * VC) sv[idx] = rv[e];
    }
    if (tid < TC) sb[tid] = rb;
  };

  if (n > 0) fetch(0);
  for (int t0 = 0; t0 < n; t0 += TC) {
    __syncthreads();   // the previous tokens have been used
    stage();
    __syncthreads();
    if (t0 + TC < n) fetch(t0 + TC);
    const int tn = min(TC, n - t0);
    for (int t = 0; t < tn; ++t) {
      float kk[R], acc[CPT];
      const float4* k4 = reinterpret_cast<const float4*>(sk + t * ROW + rg * SEG);
      const float4* a4 = reinterpret_cast<const float4*>(sa + t * ROW + rg * SEG);
      const float4* q4 = reinterpret_cast<const float4*>(sq + t * ROW + rg * SEG);
#pragma unroll
      for (int c = 0; c < CPT; ++c) acc[c] = 0.f;
#pragma unroll
      for (int r = 0; r < R / 4; ++r) {
        const float4 kv = k4[r], av = a4[r];
        const float ks[4] = {kv.x, kv.y, kv.z, kv.w}, as[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          kk[4 * r + j] = ks[j];
#pragma unroll
          for (int c = 0; c < CPT; ++c) {
            st[4 * r + j][c] *= as[j];
            acc[c] = fmaf(st[4 * r + j][c], ks[j], acc[c]);
          }
        }
      }
#pragma unroll
      for (int d = CL; d < 32; d <<= 1)
#pragma unroll
        for (int c = 0; c < CPT; ++c) acc[c] += __shfl_xor_sync(0xffffffffu, acc[c], d);
      const float beta = sb[t];
      float u[CPT], oa[CPT];
#pragma unroll
      for (int c = 0; c < CPT; ++c) {
        u[c] = beta * (sv[t * VC + c0 + c] - beta * acc[c]);
        oa[c] = 0.f;
      }
#pragma unroll
      for (int r = 0; r < R / 4; ++r) {
        const float4 qv = q4[r];
        const float qs[4] = {qv.x, qv.y, qv.z, qv.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int c = 0; c < CPT; ++c) {
            st[4 * r + j][c] = fmaf(kk[4 * r + j], u[c], st[4 * r + j][c]);
            oa[c] = fmaf(st[4 * r + j][c], qs[j], oa[c]);
          }
      }
#pragma unroll
      for (int d = CL; d < 32; d <<= 1)
#pragma unroll
        for (int c = 0; c < CPT; ++c) oa[c] += __shfl_xor_sync(0xffffffffu, oa[c], d);
      if (rg == 0) stc<CPT>(o + (long long)(t0 + t) * p.H * K + c0, oa);
    }
  }
  float* s1 = p.s1 + (bh * K + rg * R) * K + col;
#pragma unroll
  for (int r = 0; r < R; ++r) stc<CPT>(s1 + r * K, st[r]);
  // tokens past the sequence's count have output 0
  for (int idx = tid; idx < (p.S - n) * VC; idx += THREADS)
    o[(long long)(n + idx / VC) * p.H * K + idx % VC] = 0.f;
}

template <typename T, int K, int RG, int CPT, int VC, int TC>
void launch_rec(const RecParams& p) {
  const long long blocks = (long long)p.B * p.H * (K / VC);
  HB_CHECK(blocks < (1ll << 31), "kda_recurrent: too many (sequence, head) pairs");
  kda_recurrent_kernel<T, K, RG, CPT, VC, TC><<<(unsigned)blocks, VC / CPT * RG, 0, cur_stream()>>>(p);
  HB_CUDA_CHECK(cudaGetLastError());
}

template <typename T>
void dispatch_rec(const RecParams& p, int K) {
  if (p.S <= 8) {   // bound by the state's traffic: wide columns, one pass over few tokens
    if (K == 16) launch_rec<T, 16, 4, 2, 16, 2>(p);
    else if (K == 32) launch_rec<T, 32, 4, 4, 32, 2>(p);
    else if (K == 64) launch_rec<T, 64, 4, 4, 64, 2>(p);
    else launch_rec<T, 128, 8, 4, 64, 2>(p);
  } else {
    if (K == 16) launch_rec<T, 16, 4, 1, 16, 16>(p);
    else if (K == 32) launch_rec<T, 32, 4, 1, 32, 16>(p);
    else if (K == 64) launch_rec<T, 64, 4, 1, 32, 16>(p);
    else launch_rec<T, 128, 8, 1, 32, 8>(p);
  }
}

Row3 row3(const torch::Tensor& t) { return {t.stride(0), t.stride(1), t.stride(2)}; }

}  // namespace

// q, k, v [B, S, H, K] (fp32 or bf16), g like them in fp32, beta [B, S, H] fp32,
// s0 [B or 1, H, K, K] fp32 or none -> o [B, S, H, K] and s1 [B, H, K, K], both
// fp32 and contiguous.
std::tuple<torch::Tensor, torch::Tensor> kda_recurrent(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor g,
                                                       torch::Tensor beta, c10::optional<double> scale, OptTensor s0,
                                                       OptTensor counts) {
  const auto dev = q.device();
  const c10::cuda::CUDAGuard guard(dev);
  need(q.dim() == 4 && k.sizes() == q.sizes() && v.sizes() == q.sizes() && g.sizes() == q.sizes() &&
           beta.sizes() == q.sizes().slice(0, 3),
       "kda_recurrent: q, k, v, g [B, S, H, K] and beta [B, S, H]");
  need(k.device() == dev && v.device() == dev && g.device() == dev && beta.device() == dev,
       "kda_recurrent: all inputs on one device");
  need(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() &&
           (q.scalar_type() == at::kFloat || q.scalar_type() == at::kBFloat16) && g.scalar_type() == at::kFloat &&
           beta.scalar_type() == at::kFloat,
       "kda_recurrent: fp32 or bf16 q, k, v; fp32 g and beta");
  const int64_t B = q.size(0), S = q.size(1), H = q.size(2), K = q.size(3);
  need(K == 16 || K == 32 || K == 64 || K == 128, "kda_recurrent: head dim 16, 32, 64 or 128");
  if (s0)
    need(s0->dim() == 4 && (s0->size(0) == 1 || s0->size(0) == B) && s0->size(1) == H && s0->size(2) == K &&
             s0->size(3) == K && s0->device() == dev && s0->scalar_type() == at::kFloat,
         "kda_recurrent: state [B or 1, H, K, K] fp32 on the inputs' device");
  for (const auto& t : {q, k, v, g, beta}) need(!wants_grad(t), "kda_recurrent has no backward: call it under torch.no_grad()");
  need(!s0 || !wants_grad(*s0), "kda_recurrent has no backward: call it under torch.no_grad()");
  if (counts) counts = whole(*counts, B, dev, "kda_recurrent: counts, B whole numbers on the inputs' device");
  const auto opt = q.options().dtype(at::kFloat);
  torch::Tensor o = torch::empty({B, S, H, K}, opt), s1 = torch::empty({B, H, K, K}, opt);
  if (B * H == 0) return {o, s1};
  const auto rows = [](const torch::Tensor& t) { return t.stride(3) == 1 ? t : t.contiguous(); };
  q = rows(q), k = rows(k), v = rows(v), g = rows(g);
  if (s0) {   // 16-byte loads of contiguous states; a broadcast over the batch stays one
    const auto z = s0->stride(0) == 0 && B > 1 ? s0->narrow(0, 0, 1) : *s0;
    const bool ok = z.select(0, 0).is_contiguous() && reinterpret_cast<uintptr_t>(z.data_ptr()) % 16 == 0 &&
                    (z.size(0) == 1 || z.stride(0) % 4 == 0);
    s0 = ok ? z : z.clone(at::MemoryFormat::Contiguous);
  }
  RecParams p{};
  p.q = q.data_ptr(), p.k = k.data_ptr(), p.v = v.data_ptr();
  p.g = g.data_ptr<float>(), p.beta = beta.data_ptr<float>();
  p.qs = row3(q), p.ks = row3(k), p.vs = row3(v), p.gs = row3(g), p.bs = row3(beta);
  p.s0 = s0 ? s0->data_ptr<float>() : nullptr;
  p.s0_b = s0 && s0->size(0) > 1 ? s0->stride(0) : 0;
  p.s1 = s1.data_ptr<float>(), p.o = o.data_ptr<float>();
  p.counts = counts ? counts->data_ptr<int>() : nullptr;
  p.B = (int)B, p.S = (int)S, p.H = (int)H;
  p.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)K));
  p.status = status_ptr();
  if (q.scalar_type() == at::kFloat) dispatch_rec<float>(p, (int)K);
  else dispatch_rec<__nv_bfloat16>(p, (int)K);
  return {o, s1};
}

}  // namespace hb
