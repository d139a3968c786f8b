// One query token per sequence over the slots of the heavy-hitter cache, with the weights
// added to the slots' masses.
//
//   o = sum_n p_n v_n,  p_n = exp(c q . k_n - lse),  mass_n += sum over the group's heads of p_n
//
// HBM-bound: K and V are read once (2 D elements a slot), everything else is small.  A
// (sequence, kv head) is a cluster of CTAs that cut its slots; a warp takes 16 slots at a
// time straight from global memory into mma.sync fragments: the contraction index of
// S^T = K Q^T is permuted the same way in K and q, so that a lane's fragments are 16-byte
// pieces of a row, and for O^T = V^T P^T the output channels are permuted instead, with
// pairs of slots joined by byte permutes.  No shared-memory stage, no barrier in the loop.
// The final weights need the whole row's lse, so the scores stay in shared memory (in the
// workspace when a part of the slots is too long for that) until the cluster has merged its
// (o, m, l) over distributed shared memory; every CTA then updates the masses of its own
// slots.  One launch, no atomics: the sums have a fixed order.
// P is split into hi + lo 16-bit parts (to ~2^-16), so o carries its own rounding only.
#include <cooperative_groups.h>

#include <cstdio>
#include <type_traits>

#include "launchers.cuh"
#include "sparse_attention_mma.cuh"
#include "umma.cuh"

namespace cg = cooperative_groups;

namespace linattn {

namespace {

struct HeavyAttendArgs {
  const uint4* k;
  const uint4* v;
  float* mass;
  const int32_t* seen;
  const void* q;
  void* out;
  int64_t qb, qh, ob, oh;
  int H, M, G;
  float scale_log2;
  int accumulate;
  float* scores;     // workspace (B, H, 8 NT, M), or NULL: scores in shared memory
  int part_max;      // slots of a CTA's part at most (a multiple of 16)
};

constexpr int ATT_WARPS = 8;

template <int NT>
constexpr int attend_fixed_smem(int D) {  // floats: per-warp o, the CTA's o, (m, l) per warp and of the CTA
  return ATT_WARPS * 8 * NT * D + 8 * NT * D + 2 * ATT_WARPS * 8 * NT + 2 * 8 * NT;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * ATT_WARPS, NT == 1 ? 2 : 1) heavy_attend_kernel(const HeavyAttendArgs a) {
  using M = MmaOp<T>;
  constexpr int PIECES = D / 8;        // 16-byte pieces of a row
  constexpr int KJ = D / 32;           // pieces of a K row per lane
  constexpr int VJ = D / 64;           // pieces of a V row per lane
  constexpr int MT = D / 16;           // 16-channel tiles of O^T
  constexpr int HN = 8 * NT;           // head columns
  extern __shared__ __align__(16) float dsm[];
  float* o_warp = dsm;                               // [ATT_WARPS][HN][D]
  float* o_cta = o_warp + ATT_WARPS * HN * D;        // [HN][D]
  float* ml_warp = o_cta + HN * D;                   // [2][ATT_WARPS][HN]
  float* ml_cta = ml_warp + 2 * ATT_WARPS * HN;      // [2][HN]
  float* sc_smem = ml_cta + 2 * HN;                  // [HN][part_max]
  cg::cluster_group cluster = cg::this_cluster();
  const int cl = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int unit = blockIdx.x / cl, h = unit % a.H, b = unit / a.H;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tig = lane & 3;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int count = min(a.seen[b], a.M);
  const int part = ((count + 16 * cl - 1) / (16 * cl)) * 16;
  const int lo = min(count, rank * part), hi = min(count, lo + part);
  const uint4* kp = a.k + static_cast<int64_t>(unit) * a.M * PIECES;
  const uint4* vp = a.v + static_cast<int64_t>(unit) * a.M * PIECES;
  float* mass = a.mass + static_cast<int64_t>(unit) * a.M;
  const int64_t sc_stride = a.scores ? a.M : a.part_max;
  float* sc = a.scores ? a.scores + static_cast<int64_t>(unit) * HN * a.M + lo : sc_smem;

  for (int h0 = 0; h0 < a.G; h0 += HN) {  // groups of more than HN heads: HN at a time
    const int heads = min(HN, a.G - h0);
    // q of head g: the same permuted channels as the K fragments
    uint4 q[NT][KJ];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
        const int head = t * 8 + g;
        q[t][j] = make_uint4(0u, 0u, 0u, 0u);
        if (head < heads)
          q[t][j] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.qb +
                                                    (static_cast<int64_t>(h) * a.G + h0 + head) * a.qh + (tig + 4 * j) * 8);
      }
    float acc[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int e = 0; e < MT; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][e][i] = 0.f;
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
    }
    uint4 kf[KJ][2], vf[VJ][4];
    auto load_k = [&](int base) {
      const int r0 = min(base + g, hi - 1), r1 = min(base + g + 8, hi - 1);
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
        kf[j][0] = __ldg(kp + static_cast<int64_t>(r0) * PIECES + tig + 4 * j);
        kf[j][1] = __ldg(kp + static_cast<int64_t>(r1) * PIECES + tig + 4 * j);
      }
    };
    auto load_v = [&](int base) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int r = min(base + 2 * tig + (x & 1) + 8 * (x >> 1), hi - 1);
#pragma unroll
        for (int j = 0; j < VJ; ++j) vf[j][x] = __ldg(vp + static_cast<int64_t>(r) * PIECES + g + 8 * j);
      }
    };
    int base = lo + 16 * warp;
    if (base < hi) {
      load_k(base);
      load_v(base);
    }
    for (; base < hi; base += 16 * ATT_WARPS) {
      const int next = base + 16 * ATT_WARPS;
      float s[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
        const uint32_t f0[4] = {kf[j][0].x, kf[j][1].x, kf[j][0].y, kf[j][1].y};
        const uint32_t f1[4] = {kf[j][0].z, kf[j][1].z, kf[j][0].w, kf[j][1].w};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          M::mma(s[t], f0, q[t][j].x, q[t][j].y);
          M::mma(s[t], f1, q[t][j].z, q[t][j].w);
        }
      }
      if (next < hi) load_k(next);  // K of the next slots behind this tile's softmax and P V
      const bool in0 = base + g < hi, in1 = base + g + 8 < hi;
      bool grow = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = i < 2 ? in0 : in1;
          const float x = in ? s[t][i] * a.scale_log2 : -INFINITY;
          s[t][i] = x;
          const int head = t * 8 + 2 * tig + (i & 1);
          if (in && a.accumulate && head < heads) sc[head * sc_stride + (base - lo) + g + (i < 2 ? 0 : 8)] = x;
          grow |= x > m[t][i & 1] + 8.f;
        }
      }
      if (__any_sync(0xffffffffu, grow)) {  // the running maximum moves only past a margin of 2^8
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = fmaxf(s[t][c], s[t][c + 2]);
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            mx = fmaxf(mx, m[t][c]);
            const float f = m[t][c] == -INFINITY ? 0.f : ex2_approx(m[t][c] - mx);
            m[t][c] = mx;
            l[t][c] *= f;
#pragma unroll
            for (int e = 0; e < MT; ++e) {
              acc[t][e][c] *= f;
              acc[t][e][c + 2] *= f;
            }
          }
      }
      uint32_t bh[NT][2], bl[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float z0 = m[t][0] == -INFINITY ? 0.f : m[t][0], z1 = m[t][1] == -INFINITY ? 0.f : m[t][1];
        const float p0 = ex2_approx(s[t][0] - z0), p1 = ex2_approx(s[t][1] - z1);
        const float p2 = ex2_approx(s[t][2] - z0), p3 = ex2_approx(s[t][3] - z1);
        l[t][0] += p0 + p2;
        l[t][1] += p1 + p3;
        const uint32_t h01 = M::pack(p0, p1), h23 = M::pack(p2, p3);
        const float2 r01 = M::unpack(h01), r23 = M::unpack(h23);
        bh[t][0] = movmatrix_t(h01);
        bh[t][1] = movmatrix_t(h23);
        bl[t][0] = movmatrix_t(M::pack(p0 - r01.x, p1 - r01.y));
        bl[t][1] = movmatrix_t(M::pack(p2 - r23.x, p3 - r23.y));
      }
      // O^T: rows g / g + 8 of tile e are channel e of pieces g and g + 8 (D = 128), or
      // channels e and e + 4 of piece g (D = 64)
#pragma unroll
      for (int e = 0; e < MT; ++e) {
        const int e0 = e, e1 = VJ == 2 ? e : e + MT, j1 = VJ == 2 ? VJ - 1 : 0;
        auto word = [&](const uint4& w, int c) { return c < 2 ? w.x : c < 4 ? w.y : c < 6 ? w.z : w.w; };
        auto join = [&](int j, int c, int x) {
          return __byte_perm(word(vf[j][x], c), word(vf[j][x + 1], c), (c & 1) ? 0x7632 : 0x5410);
        };
        const uint32_t f[4] = {join(0, e0, 0), join(j1, e1, 0), join(0, e0, 2), join(j1, e1, 2)};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          M::mma(acc[t][e], f, bh[t][0], bh[t][1]);
          M::mma(acc[t][e], f, bl[t][0], bl[t][1]);
        }
      }
      if (next < hi) load_v(next);
    }
    // ---- the CTA's (o, m, l)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) l[t][c] += __shfl_xor_sync(0xffffffffu, l[t][c], o);
        if (g == 0) {
          ml_warp[warp * HN + t * 8 + 2 * tig + c] = m[t][c];
          ml_warp[(ATT_WARPS + warp) * HN + t * 8 + 2 * tig + c] = l[t][c];
        }
#pragma unroll
        for (int e = 0; e < MT; ++e)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int ch = VJ == 2 ? (g + 8 * r) * 8 + e : g * 8 + e + 4 * r;
            o_warp[(warp * HN + t * 8 + 2 * tig + c) * D + ch] = acc[t][e][c + 2 * r];
          }
      }
    __syncthreads();
    for (int i = tid; i < HN * D; i += 32 * ATT_WARPS) {
      const int head = i / D;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < ATT_WARPS; ++w) mx = fmaxf(mx, ml_warp[w * HN + head]);
      float o = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < ATT_WARPS; ++w) {
        // a warp without slots (m = -inf, l = 0) is left out; one whose scores are all NaN
        // (m = -inf, l = NaN) is not
        const float mw = ml_warp[w * HN + head], lw = ml_warp[(ATT_WARPS + w) * HN + head];
        const float f = mw == -INFINITY ? lw : ex2_approx(mw - mx);
        if (f != 0.f) {
          o += f * o_warp[w * HN * D + i];
          sum += f * lw;
        }
      }
      o_cta[i] = o;
      if (i % D == 0) {
        ml_cta[head] = mx;
        ml_cta[HN + head] = sum;
      }
    }
    cluster.sync();
    // ---- merge over the cluster; this CTA writes its share of the outputs
    float* lse2 = ml_warp;  // [HN] maximum, then [HN] 1 / sum (ml_warp is no longer read)
    if (tid < HN) {
      float mx = -INFINITY, sum = 0.f;
      for (int r = 0; r < cl; ++r) mx = fmaxf(mx, cluster.map_shared_rank(ml_cta, r)[tid]);
      for (int r = 0; r < cl; ++r) {
        const float* o = cluster.map_shared_rank(ml_cta, r);
        sum += o[tid] == -INFINITY ? o[HN + tid] : ex2_approx(o[tid] - mx) * o[HN + tid];
      }
      lse2[tid] = mx == -INFINITY ? 0.f : mx;
      lse2[HN + tid] = sum != 0.f ? 1.f / sum : 0.f;
    }
    __syncthreads();
    for (int i = rank * 32 * ATT_WARPS + tid; i < heads * D; i += cl * 32 * ATT_WARPS) {
      const int head = i / D;
      float o = 0.f;
      for (int r = 0; r < cl; ++r) {
        const float* ml = cluster.map_shared_rank(ml_cta, r);
        const float f = ml[head] == -INFINITY ? ml[HN + head] : ex2_approx(ml[head] - lse2[head]);
        if (f != 0.f) o += f * cluster.map_shared_rank(o_cta, r)[i];
      }
      store_any(a.out, b * a.ob + (static_cast<int64_t>(h) * a.G + h0 + head) * a.oh + i % D,
                std::is_same<T, __half>::value ? LINATTN_F16 : LINATTN_BF16, o * lse2[HN + head]);
    }
    if (a.accumulate)
      for (int n = tid; n < hi - lo; n += 32 * ATT_WARPS) {
        float w = 0.f;
        for (int e = 0; e < heads; ++e) w += ex2_approx(sc[e * sc_stride + n] - lse2[e]) * lse2[HN + e];
        mass[lo + n] += w;
      }
    cluster.sync();  // o_cta and ml_cta are read by the other CTAs; the buffers are free again
  }
}

int attend_fail(int code, const char* what) {
  char msg[256];
  snprintf(msg, sizeof(msg), "heavy_attend: %s", what);
  return set_error(code, msg);
}

struct AttendPlan {
  int nt, cl, part, smem;
  bool global_scores;
};

constexpr int ATT_SMEM_SCORES = 64 * 1024;  // scores of a part kept in shared memory at most

// Cluster size: enough CTAs for about four rounds of the GPU's 296 (two to an SM), with at
// least 128 slots each (16 for each warp).
AttendPlan attend_plan(int64_t units, int64_t G, int64_t M, int D) {
  AttendPlan p;
  p.nt = G > 8 ? 2 : 1;
  p.cl = 1;
  while (p.cl < 8 && units * p.cl < 592 && M > 128 * p.cl) p.cl *= 2;
  p.part = static_cast<int>((M + 16 * p.cl - 1) / (16 * p.cl)) * 16;
  const int64_t heads = 8 * p.nt;
  const int64_t scores = heads * p.part * 4;
  p.global_scores = scores > ATT_SMEM_SCORES;
  const int fixed = (p.nt == 1 ? attend_fixed_smem<1>(D) : attend_fixed_smem<2>(D)) * 4;
  p.smem = fixed + (p.global_scores ? 0 : static_cast<int>(scores));
  return p;
}

template <typename T, int D, int NT>
cudaError_t launch_attend(const HeavyAttendArgs& a, const AttendPlan& p, int64_t units, cudaStream_t st) {
  auto kern = heavy_attend_kernel<T, D, NT>;
  static int allowed[64] = {};
  cudaError_t e = allow_smem(kern, p.smem, allowed);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(static_cast<unsigned>(units * p.cl));
  cfg.blockDim = dim3(32 * ATT_WARPS);
  cfg.dynamicSmemBytes = static_cast<size_t>(p.smem);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.cl);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

template <typename T>
cudaError_t dispatch_attend(const HeavyAttendArgs& a, const AttendPlan& p, int D, int64_t units, cudaStream_t st) {
  if (D == 128) return p.nt == 1 ? launch_attend<T, 128, 1>(a, p, units, st) : launch_attend<T, 128, 2>(a, p, units, st);
  return p.nt == 1 ? launch_attend<T, 64, 1>(a, p, units, st) : launch_attend<T, 64, 2>(a, p, units, st);
}

}  // namespace

}  // namespace linattn

using namespace linattn;

extern "C" int64_t linattn_heavy_attend_workspace(int64_t batch, int64_t Hq, int64_t Hkv, int64_t budget) {
  if (batch < 1 || Hkv < 1 || Hq < 1 || budget < 1) return 0;
  const AttendPlan p = attend_plan(batch * Hkv, Hq / Hkv, budget, 128);
  return p.global_scores ? batch * Hkv * 8 * p.nt * budget * 4 : 0;
}

extern "C" int linattn_heavy_attend(const linattn_heavy_t* cache, const void* q, int64_t Hq, const int64_t* q_strides,
                                    float scale, int32_t accumulate, void* out, const int64_t* out_strides,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
  if (!cache || !cache->k || !cache->v || !cache->mass || !cache->seen || !q || !out || !q_strides || !out_strides)
    return attend_fail(LINATTN_EINVAL, "NULL pointer");
  if (cache->dtype != LINATTN_F16 && cache->dtype != LINATTN_BF16)
    return attend_fail(LINATTN_EUNSUPPORTED, "f16 or bf16 caches");
  if (cache->head_dim != 64 && cache->head_dim != 128) return attend_fail(LINATTN_EUNSUPPORTED, "head_dim must be 64 or 128");
  if (cache->batch < 1 || cache->n_kv_heads < 1 || cache->budget < 1 || cache->budget > (1 << 24))
    return attend_fail(LINATTN_EINVAL, "batch, n_kv_heads and budget must be > 0 (budget <= 2^24)");
  if (Hq < 1 || Hq % cache->n_kv_heads) return attend_fail(LINATTN_EINVAL, "H_q must be a multiple of H_kv");
  if (!(scale > 0.f) || scale > 1e30f) return attend_fail(LINATTN_EINVAL, "scale must be positive and finite");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache->k) | reinterpret_cast<uintptr_t>(cache->v)) % 16 ||
      q_strides[0] % 8 || q_strides[1] % 8)
    return attend_fail(LINATTN_EINVAL, "q, K and V rows must be 16-byte aligned");
  const int64_t units = static_cast<int64_t>(cache->batch) * cache->n_kv_heads;
  const int64_t G = Hq / cache->n_kv_heads;
  const AttendPlan p = attend_plan(units, G, cache->budget, cache->head_dim);
  if (units * p.cl >= (int64_t(1) << 31) || G > 1024) return attend_fail(LINATTN_EUNSUPPORTED, "too many heads");
  if (p.global_scores && accumulate && (!workspace || workspace_bytes < units * 8 * p.nt * cache->budget * 4))
    return attend_fail(LINATTN_EINVAL, "workspace too small");
  HeavyAttendArgs a;
  a.k = static_cast<const uint4*>(cache->k);
  a.v = static_cast<const uint4*>(cache->v);
  a.mass = cache->mass;
  a.seen = cache->seen;
  a.q = q;
  a.out = out;
  a.qb = q_strides[0];
  a.qh = q_strides[1];
  a.ob = out_strides[0];
  a.oh = out_strides[1];
  a.H = cache->n_kv_heads;
  a.M = cache->budget;
  a.G = static_cast<int>(G);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.accumulate = accumulate ? 1 : 0;
  a.scores = p.global_scores && accumulate ? static_cast<float*>(workspace) : nullptr;
  a.part_max = p.part;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = cache->dtype == LINATTN_F16 ? dispatch_attend<__half>(a, p, cache->head_dim, units, st)
                                                    : dispatch_attend<__nv_bfloat16>(a, p, cache->head_dim, units, st);
  return e == cudaSuccess ? LINATTN_OK : attend_fail(LINATTN_ECUDA, cudaGetErrorString(e));
}
