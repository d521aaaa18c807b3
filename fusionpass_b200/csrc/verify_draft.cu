// Verification of drafted tokens against the target's probabilities, from given random
// numbers (include/fpkern.h states the walk).
//
// At a node the drafts that failed change the target's probabilities t to
//   r_k = max(r_k-1 - m_k-1 q, 0),  r_0 = t,  m_0 = 1,  m_k = sum r_k,
// with one and the same q for all children of a node, q >= 0, so that
//   r_k = max(t - (m_0 + ... + m_k-1) q, 0):
// a number M is all that is kept of the failures, and r is made anew from t and q wherever it is
// read.  Without draft probabilities r is t with the failed tokens left out.  Sums and
// comparisons are in 64 bits: a running sum over 10^5 values meets 10^5 borders, and one in
// 32 bits picks another token at some of them.
//
// One cluster a sequence (1 to 8 CTAs): warp w of CTA c holds a stretch of the vocabulary.  What the
// children's tests need is fetched ahead for the whole tree, so that a walk without failures costs
// no more than its last row.  A failure, or the end, takes a pass over a row: each warp's sum in a
// fixed order, the CTAs' sums handed round through shared memory.  For the last token the CTA whose
// sums hold the border sums its warp's stretch again in steps of 32, and a warp looks through one.
// Bound by the latency of those passes for few sequences, by reading the rows for many.
#include <cuda_runtime.h>

#include <cstring>

#include "internal.h"
#include "score_common.cuh"

namespace fpk {
namespace verify {
namespace {

constexpr int kWarps = 16;
constexpr int kThreads = 32 * kWarps;
constexpr int kNodes = FPK_TREE_MAX_NODES;
constexpr int kMaxCtas = 8;
constexpr int kMaxSteps = FPK_VERIFY_MAX_VOCAB / 32 / kWarps / kMaxCtas;  // of 32 tokens, in a warp's stretch
constexpr int kAhead = 8;   // steps of 32 tokens whose values are asked for at once
constexpr int kAhead4 = 4;  // steps of 128

struct Smem {
  int parent[kNodes], token[kNodes];
  float t_at[kNodes], q_at[kNodes], uniform[kNodes];
  int failed[kNodes];            // tokens left out at this node (without draft)
  double warp_sum[kWarps];
  double cta_sum[2][kMaxCtas];   // written by the cluster's CTAs, in turn
  double step_sum[kMaxSteps];
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}
__device__ __forceinline__ void store_remote(double* p, uint32_t rank, double v) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(v) : "memory");
}
__device__ __forceinline__ double warp_total(double v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// What the walk reads at a node.  A probability that is negative or NaN counts as 0 (fmax).
struct Row {
  const float* t;
  const float* q;  // null: without draft, or nothing has failed here
  double m;        // M
  int n_failed;    // tokens left out
};
__device__ __forceinline__ double left_of(const Row& r, float t, float q) {
  return fmax(__dsub_rn(static_cast<double>(t), __dmul_rn(r.m, static_cast<double>(q))), 0.0);
}
// r of steps x0, x0 + 1, ... of 32 tokens from `from`, this lane's token of each; 0 beyond `end`
template <int N>
__device__ __forceinline__ void values(const Row& r, const int* failed, int from, int end, int lane, double* out) {
  float t[N], q[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int x = from + 32 * i + lane;
    t[i] = x < end ? __ldg(r.t + x) : 0.0f;
    q[i] = r.q && x < end ? fmaxf(__ldg(r.q + x), 0.0f) : 0.0f;
  }
  for (int k = 0; k < r.n_failed; ++k) {
    const int x = failed[k] - from - lane;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (x == 32 * i) t[i] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = left_of(r, t[i], q[i]);
}

__global__ void __launch_bounds__(kThreads, 2) verify_kernel(const __grid_constant__ fpk_verify_desc p, int stretch, int wide) {
  __shared__ Smem sm;
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  const int ctas = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
  const int64_t b = blockIdx.x / ctas;
  cluster_arrive();  // waited for below: every CTA runs before the first writes to another
  score::grid_wait();
  const int n = p.tree_lens ? min(max(__ldg(p.tree_lens + b), 0), p.nodes) : p.nodes;
  const float* target = p.target + b * p.target_strides[0];
  const float* draft = p.draft ? p.draft + b * p.draft_strides[0] : nullptr;
  for (int i = tid; i < n; i += kThreads) {
    int parent = __ldg(p.parents + b * p.parents_stride + i);
    const int token = __ldg(p.tokens + b * p.tokens_stride + i);
    if (i == 0 || parent < 0 || parent >= i || token < 0 || token >= p.vocab) parent = -1;  // no child of any node
    sm.parent[i] = parent;
    sm.token[i] = token;
    sm.uniform[i] = __ldg(p.uniform + b * p.uniform_stride + i);
    sm.t_at[i] = parent >= 0 ? __ldg(target + parent * p.target_strides[1] + token) : 0.0f;
    sm.q_at[i] = parent >= 0 && draft ? fmaxf(__ldg(draft + parent * p.draft_strides[1] + token), 0.0f) : 1.0f;
  }
  int* path = p.path + b * p.nodes;
  if (rank == 0)
    for (int i = tid; i < p.nodes; i += kThreads) path[i] = i == 0 && n > 0 ? 0 : -1;
  __syncthreads();
  cluster_wait();
  if (n == 0) {  // the same for the whole cluster
    if (rank == 0 && tid == 0) {
      p.counts[b] = 0;
      p.next[b] = -1;
    }
    return;
  }
  const int from = (rank * kWarps + warp) * stretch;  // below 2^31: the vocabulary rounded up
  const int end = min(from + stretch, p.vocab);
  int turn = 0;
  double total = 0.0;
  // the sum of r over the vocabulary, the same in every thread of the cluster
  const auto sum = [&](const Row& r) {
    double v = 0.0;
    int mine = 0;  // tokens left out in this warp's stretch: most have none
    for (int k = lane; k < r.n_failed; k += 32) mine |= sm.failed[k] >= from && sm.failed[k] < end;
    Row w = r;
    if (!__any_sync(0xffffffffu, mine)) w.n_failed = 0;
    if (wide && w.n_failed == 0) {  // four tokens a lane and load
      for (int x = from; x < end; x += 128 * kAhead4) {
        float4 t[kAhead4], q[kAhead4];
#pragma unroll
        for (int i = 0; i < kAhead4; ++i) {
          const int at = x + 128 * i + 4 * lane;
          const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          t[i] = at < end ? __ldg(reinterpret_cast<const float4*>(w.t + at)) : none;
          q[i] = w.q && at < end ? __ldg(reinterpret_cast<const float4*>(w.q + at)) : none;
        }
#pragma unroll
        for (int i = 0; i < kAhead4; ++i) {
          v += left_of(w, t[i].x, fmaxf(q[i].x, 0.0f)) + left_of(w, t[i].y, fmaxf(q[i].y, 0.0f));
          v += left_of(w, t[i].z, fmaxf(q[i].z, 0.0f)) + left_of(w, t[i].w, fmaxf(q[i].w, 0.0f));
        }
      }
    } else {
      for (int x = from; x < end; x += 32 * kAhead) {
        double e[kAhead];
        values<kAhead>(w, sm.failed, x, end, lane, e);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) v += e[i];
      }
    }
    v = warp_total(v);
    if (lane == 0) sm.warp_sum[warp] = v;
    __syncthreads();
    if (tid < ctas) {
      double s = 0.0;
      for (int w2 = 0; w2 < kWarps; ++w2) s += sm.warp_sum[w2];
      store_remote(&sm.cta_sum[turn][rank], static_cast<uint32_t>(tid), s);
    }
    cluster_sync();
    total = 0.0;
    for (int c = 0; c < ctas; ++c) total += sm.cta_sum[turn][c];
    turn ^= 1;
  };

  int at = 0, count = 1, seen = 0;  // nodes up to `seen` have been looked at
  bool fresh = true;                // the sums are not those of the row as it is
  double m = 1.0;
  Row row{target, nullptr, 0.0, 0};
  for (;;) {
    // the next child of `at`, in order
    int x = -1;
    for (int c = (seen + 1) & ~31; c < n && x < 0; c += 32) {
      const int i = c + lane;
      const uint32_t hit = __ballot_sync(0xffffffffu, i > seen && i < n && sm.parent[i] == at);
      if (hit) x = c + __ffs(hit) - 1;
    }
    if (x < 0) break;
    seen = x;
    const int token = sm.token[x];
    double r = left_of(row, sm.t_at[x], row.q ? sm.q_at[x] : 0.0f);
    if (row.n_failed > 0) {
      int out = 0;
      for (int k = lane; k < row.n_failed; k += 32) out |= sm.failed[k] == token;
      if (__any_sync(0xffffffffu, out)) r = 0.0;
    }
    const double need = __dmul_rn(static_cast<double>(sm.uniform[x]) * static_cast<double>(sm.q_at[x]), m);
    if (need < r) {
      if (rank == 0 && tid == 0) path[count] = x;
      ++count;
      at = x;
      m = 1.0;
      fresh = true;
      row = Row{target + at * p.target_strides[1], nullptr, 0.0, 0};
      __syncthreads();  // the list of failures is read no more
      continue;
    }
    if (draft) {
      row.q = draft + at * p.draft_strides[1];
      row.m += m;
    } else {
      __syncthreads();  // it has been read as it was
      if (tid == 0) sm.failed[row.n_failed] = token;
      ++row.n_failed;
      __syncthreads();
    }
    sum(row);
    m = total;
    fresh = false;
  }
  if (fresh) sum(row);
  int next = -1;
  if (total > 0.0 && total < INFINITY) {
    const double u = fmin(fmax(static_cast<double>(sm.uniform[0]), 0.0), 1.0 - 0x1p-24);
    const double border = __dmul_rn(u, total);
    // the CTA, then its warp, whose sums pass the border; where roundings leave no warp, or step, that
    // does, the last with any (the CTAs' sums make up the total in this order: one of them does)
    double base = 0.0;
    int cta = 0;
    while (cta + 1 < ctas && !(base + sm.cta_sum[turn ^ 1][cta] > border)) base += sm.cta_sum[turn ^ 1][cta++];
    if (cta == rank) {
      int w = -1;
      double wbase = base;
      for (int i = 0; i < kWarps; ++i) {
        const double s = sm.warp_sum[i];
        if (s > 0.0) {
          w = i;
          wbase = base;
        }
        if (base + s > border) break;
        base += s;
      }
      // its stretch in steps of 32, shared by the warps
      const int wfrom = (rank * kWarps + w) * stretch, wend = min(wfrom + stretch, p.vocab);
      const int steps = (wend - wfrom + 31) / 32;
      for (int i = warp; i < steps; i += kWarps) {
        double e[1];
        values<1>(row, sm.failed, wfrom + 32 * i, wend, lane, e);
        const double s = warp_total(e[0]);
        if (lane == 0) sm.step_sum[i] = s;
      }
      __syncthreads();
      if (warp == 0) {
        int step = -1;
        double sbase = wbase;
        for (int i = 0; i < steps; ++i) {
          const double s = sm.step_sum[i];
          if (s > 0.0) {
            step = i;
            sbase = wbase;
          }
          if (wbase + s > border) break;
          wbase += s;
        }
        double e[1];
        values<1>(row, sm.failed, wfrom + 32 * step, wend, lane, e);
        double run = e[0];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const double o = __shfl_up_sync(0xffffffffu, run, off);
          if (lane >= off) run += o;
        }
        const uint32_t some = __ballot_sync(0xffffffffu, e[0] > 0.0);
        const uint32_t past = __ballot_sync(0xffffffffu, e[0] > 0.0 && sbase + run > border);
        next = wfrom + 32 * step + (past ? __ffs(past) - 1 : 31 - __clz(some));
        if (lane == 0) p.next[b] = next;
      }
    }
  } else if (rank == 0 && tid == 0) {
    p.next[b] = -1;
  }
  if (rank == 0 && tid == 0) p.counts[b] = count;
  cluster_sync();  // no CTA goes while another may still write to it
}

int check(const fpk_verify_desc* d) {
  if (!d || d->size != sizeof(fpk_verify_desc) || d->version != FPK_ABI_VERSION) return FPK_ERR_INVALID;
  if (d->batch < 0 || d->nodes < 1 || d->vocab < 1) return FPK_ERR_INVALID;
  if (d->nodes > FPK_TREE_MAX_NODES || d->vocab > FPK_VERIFY_MAX_VOCAB || d->batch > (1 << 24))
    return FPK_ERR_UNSUPPORTED;
  if (d->batch == 0) return FPK_OK;
  if (!d->tokens || !d->parents || !d->target || !d->uniform || !d->path || !d->counts || !d->next)
    return FPK_ERR_INVALID;
  uintptr_t at = 0;
  for (const void* x : {static_cast<const void*>(d->tokens), static_cast<const void*>(d->parents),
                        static_cast<const void*>(d->target), static_cast<const void*>(d->draft),
                        static_cast<const void*>(d->uniform), static_cast<const void*>(d->tree_lens),
                        static_cast<const void*>(d->path), static_cast<const void*>(d->counts),
                        static_cast<const void*>(d->next)})
    at |= reinterpret_cast<uintptr_t>(x);
  return at % 4 ? FPK_ERR_ALIGN : FPK_OK;
}

int run(const fpk_verify_desc* d, cudaStream_t s, const DeviceInfo& dev) {
  // as many CTAs a sequence as the vocabulary fills, while all run at once (two an SM).  us with 1, 2, 4, 8 a sequence:
  // 1 of 32000 tokens 11.6, 9.2, 6.7, 6.6; 32 of 131072 82, 46, 31, 24; 16 of 50001 32, 29, 17, 15
  const int sms = dev.num_sms > 0 ? dev.num_sms : 148;
  int ctas = 1;
  while (ctas < kMaxCtas && (d->vocab > ctas * 32 * kWarps * kMaxSteps ||
                             (d->vocab > ctas * 4096 && d->batch * ctas * 2 <= 2 * sms)))
    ctas *= 2;
  // rows on 16 bytes whose length is a multiple of four tokens are read by four
  uint64_t off = reinterpret_cast<uintptr_t>(d->target) | reinterpret_cast<uintptr_t>(d->draft);
  for (int i = 0; i < 2; ++i) off |= static_cast<uint64_t>(d->target_strides[i] | (d->draft ? d->draft_strides[i] : 0)) * 4;
  const int wide = off % 16 == 0 && d->vocab % 4 == 0 ? 1 : 0;
  const int stretch = ((d->vocab + ctas * kWarps - 1) / (ctas * kWarps) + 31) / 32 * 32;
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(d->batch * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, verify_kernel, *d, stretch, wide) == cudaSuccess ? FPK_OK : FPK_ERR_CUDA;
}

}  // namespace
}  // namespace verify
}  // namespace fpk

extern "C" int fpk_verify_draft(const fpk_verify_desc* d, void* stream) {
  int rc = fpk::verify::check(d);
  if (rc != FPK_OK || d->batch == 0) return rc;
  fpk::DeviceInfo dev;
  rc = fpk::current_device_info(&dev);
  if (rc != FPK_OK) return rc;
  return fpk::verify::run(d, static_cast<cudaStream_t>(stream), dev);
}
