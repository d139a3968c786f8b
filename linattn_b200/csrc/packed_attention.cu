// Causal attention over packed sequences with grouped heads, on the 5th-generation tensor
// cores:  o_i = sum_j p_ij v_j,  p_ij = 2^(c2 q_i . k_j - lse2_i)  (log2 units), one pass over
// the keys with a running maximum and sum.
//
// A row tile is 128 / G tokens times the G heads of one kv head (128 rows, brought in by one
// 3-D tensor-map box), so that the group shares its K and V; a CTA works on two row tiles of
// one sequence with the same 128-key tiles of K and V.  Warp roles (384 threads, one CTA to
// an SM):
//   warp 0      TMA: Q once, K and V through two rings;
//   warp 1      issues tcgen05.mma: S_i = Q_i K_j^T (128 x 128, TMEM), O_i += P_i V_j with P_i
//               read from TMEM over its scores; while one tile's softmax runs, the tensor
//               cores have the other tile's P V and the next scores;
//   warp 2      clears the rows of a sequence's last V tile that belong to the next sequence
//               (0 x their Inf or NaN would reach this one);
//   warps 4-7   softmax of row tile 0, warps 8-11 of row tile 1: one thread a row.
// The running maximum moves, and O is rescaled in TMEM, only past a margin of 2^8; the sums
// are kept in fp32 from the unrounded weights, P is rounded to the inputs' 16-bit type (the
// same relative rounding as the output's).
// Bound at D = 128: a 128 x 128 tile takes 1024 clocks of the tensor cores and 1024 clocks of
// the exponential unit (16 a clock), which the two row tiles overlap.
// Few rows: the key range is cut into n_splits parts, merged by lse_combine.
#include <cstdio>
#include <type_traits>

#include "launchers.cuh"
#include "packed_tiles.cuh"
#include "sparse_attention_mma.cuh"
#include "umma.cuh"

namespace linattn {

namespace {

struct PackedArgs {
  const int32_t* cu_q;
  const int32_t* cu_k;
  int64_t Nq, Nk;
  int S, Hq, Hkv, G, tokens;  // tokens of a row tile (floor(128 / G))
  int causal;
  float scale_log2;
  void* out;
  int64_t ot, oh;
  float* lse;        // (N_q, H_q) or NULL
  int n_splits;
  float* part_o;     // (n_splits, N_q, H_q, D)
  float* part_lse;   // (n_splits, N_q, H_q)
  int32_t* status;
};

constexpr int PA_THREADS = 384;

template <int D>
struct PackedSmem {
  static constexpr int TILE = 128 * D * 2;           // Q, K or V tile
  static constexpr int KS = D == 128 ? 2 : 4;        // K ring stages
  static constexpr int VS = D == 128 ? 3 : 4;        // V ring stages
  static constexpr int BYTES = 1024 + TILE * (2 + KS + VS);
};

template <typename T, int D>
__global__ void __launch_bounds__(PA_THREADS, 1)
    packed_attention_kernel(const PackedArgs p, const __grid_constant__ CUtensorMap tmq,
                            const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv) {
  using M = MmaOp<T>;
  using SM = PackedSmem<D>;
  constexpr int KS = SM::KS, VS = SM::VS, HALVES = D / 64, TILE = SM::TILE;
  constexpr int AB = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  constexpr uint32_t IDESC_S = umma_idesc(AB, 128, 128, 0);
  constexpr uint32_t IDESC_O = umma_idesc(AB, 128, D, 1);
  extern __shared__ __align__(128) uint8_t asmem_raw[];
  uint8_t* sq = asmem_raw + ((1024 - (smem_u32(asmem_raw) & 1023)) & 1023);  // two row tiles
  uint8_t* sk = sq + 2 * TILE;
  uint8_t* sv_ring = sk + KS * TILE;
  __shared__ __align__(8) uint64_t q_full[2], k_full[KS], k_empty[KS], v_full[VS], v_empty[VS], v_ragged, s_full[2],
      p_full[2], pv_done[2], last;
  __shared__ uint32_t tmem_sh;
  __shared__ int dead;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.x % p.Hkv;
  int seq, tile;
  if (!packed_tile(p.cu_q, p.S, p.Nq, 2 * p.tokens, blockIdx.x / p.Hkv, &seq, &tile)) return;
  int q_first, lq, k_first, lk;
  bool sound = packed_range(p.cu_q, seq, p.Nq, &q_first, &lq);
  sound &= packed_range(p.cu_k, seq, p.Nk, &k_first, &lk);
  if (!sound && tid == 0) report(p.status, LINATTN_DEV_BAD_ID);
  // the last tokens of a sequence see the most keys: they come first
  tile = (lq + 2 * p.tokens - 1) / (2 * p.tokens) - 1 - tile;
  const int t0 = tile * 2 * p.tokens, shift = lk - lq;  // token t reads keys up to t + shift
  // key tiles of each row tile, and this split's share [j0, j0 + n)
  int nt[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int first = t0 + i * p.tokens, end = min(lq, first + p.tokens);
    const int keys = first >= end ? 0 : p.causal ? max(0, min(lk, end + shift)) : lk;
    nt[i] = (keys + 127) >> 7;
  }
  int j0 = 0, j1 = max(nt[0], nt[1]);
  if (p.n_splits > 1) {
    const int share = (j1 + p.n_splits - 1) / p.n_splits;
    j0 = min(j1, static_cast<int>(blockIdx.y) * share);
    j1 = min(j1, j0 + share);
  }
  const int n0 = max(0, min(nt[0], j1) - j0), n1 = max(0, min(nt[1], j1) - j0), n = max(n0, n1);
  const int boxb = p.tokens * p.G * 128;
  // the last key tile, if another sequence's rows end it
  const int ragged = (lk & 127) && j0 + n == (lk + 127) >> 7 ? n - 1 : -1;

  if (tid == 0) {
    for (int s = 0; s < KS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 128);
      mbar_init(&pv_done[s], 1);
    }
    mbar_init(&v_ragged, 1);
    mbar_init(&last, 1);
    dead = 0;
    mbar_fence_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_sh)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // columns [128 i, 128 i + 128): S / P of row tile i; [256 + 128 i, ...): O of row tile i
  const uint32_t tmem = tmem_sh;

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      int ki = 0, vi = 0;
      bool ok = true;
      auto load_q = [&](int i) {
        mbar_arrive_expect_tx(&q_full[i], boxb * HALVES);
        for (int c = 0; c < HALVES; ++c)
          tma_load_3d(sq + i * TILE + c * 16384, &tmq, 64 * c, kvh * p.G, q_first + t0 + i * p.tokens, &q_full[i]);
      };
      auto load = [&](const CUtensorMap* tm, uint8_t* ring, uint64_t* full, uint64_t* empty, int stages, int j) {
        const int st = j % stages;
        if (j >= stages) ok = mbar_wait_bounded(&empty[st], static_cast<uint32_t>((j / stages - 1) & 1));
        if (!ok || dead) return false;
        // a ragged V tile goes to warp 2 first, which passes it on
        uint64_t* bar = full == v_full && j == ragged ? &v_ragged : &full[st];
        mbar_arrive_expect_tx(bar, TILE);
        for (int c = 0; c < HALVES; ++c)
          tma_load_3d(ring + st * TILE + c * 16384, tm, 64 * c, kvh, k_first + (j0 + j) * 128, bar);
        return true;
      };
      if (n0 > 0) load_q(0);
      if (load(&tmk, sk, k_full, k_empty, KS, 0)) ki = 1;
      if (n1 > 0) load_q(1);
      for (int j = 0; j < n; ++j) {
        if (!load(&tmv, sv_ring, v_full, v_empty, VS, j)) break;
        vi = j + 1;
        if (j + 1 < n) {
          if (!load(&tmk, sk, k_full, k_empty, KS, j + 1)) break;
          ki = j + 2;
        }
      }
      if (!ok) {
        report(p.status, LINATTN_DEV_TIMEOUT);
        dead = 1;
      }
      if (dead) {  // the copies in flight land before the CTA gives up its shared memory
        if (n0 > 0) (void)mbar_wait_bounded(&q_full[0], 0, 200000000ull);
        if (n1 > 0) (void)mbar_wait_bounded(&q_full[1], 0, 200000000ull);
        for (int j = ki > KS ? ki - KS : 0; j < ki; ++j)
          (void)mbar_wait_bounded(&k_full[j % KS], static_cast<uint32_t>((j / KS) & 1), 200000000ull);
        for (int j = vi > VS ? vi - VS : 0; j < vi; ++j)
          (void)(j == ragged ? mbar_wait_bounded(&v_ragged, 0, 200000000ull)
                             : mbar_wait_bounded(&v_full[j % VS], static_cast<uint32_t>((j / VS) & 1), 200000000ull));
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && n > 0) {
      bool ok = true;
      const uint32_t qa = smem_u32(sq), ka = smem_u32(sk), va = smem_u32(sv_ring);
      auto scores = [&](int i, int j) {  // S_i of key tile j
        const uint32_t kb = ka + (j % KS) * TILE;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * 16384 + (kk & 3) * 32;
          umma_f16(tmem + i * 128, umma_desc(qa + i * TILE + off, 16, 1024), umma_desc(kb + off, 16, 1024), IDESC_S,
                   kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[i]);
      };
      auto key_tile = [&](int j) {
        ok = ok && mbar_wait_bounded(&k_full[j % KS], static_cast<uint32_t>((j / KS) & 1));
        if (ok) tc_fence_after();
      };
      key_tile(0);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (ok && (i ? n1 : n0) > 0) {
          ok = mbar_wait_bounded(&q_full[i], 0);
          if (ok) {
            tc_fence_after();
            scores(i, 0);
          }
        }
      if (ok) umma_commit(&k_empty[0]);
      for (int j = 0; ok && j < n; ++j) {
        bool v_there = false, k_there = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int ni = i ? n1 : n0;
          if (!ok || j >= ni) continue;
          if (!v_there) {
            ok = mbar_wait_bounded(&v_full[j % VS], static_cast<uint32_t>((j / VS) & 1));
            v_there = true;
          }
          ok = ok && mbar_wait_bounded(&p_full[i], static_cast<uint32_t>(j & 1));
          if (!ok) break;
          tc_fence_after();
          const uint32_t vb = va + (j % VS) * TILE;
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_f16_ts(tmem + 256 + i * 128, tmem + i * 128 + 8 * kk, umma_desc(vb + kk * 2048, 16384, 1024), IDESC_O,
                        (j > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&pv_done[i]);
          if (j + 1 < ni) {
            if (!k_there) key_tile(j + 1);
            k_there = true;
            if (ok) scores(i, j + 1);
          }
        }
        if (ok) {
          umma_commit(&v_empty[j % VS]);
          if (k_there) umma_commit(&k_empty[(j + 1) % KS]);
        }
      }
      if (!ok) {
        report(p.status, LINATTN_DEV_TIMEOUT);
        dead = 1;
      }
    }
  } else if (warp == 2) {
    if (ragged >= 0) {
      const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(&v_ragged, 0));
      if (ok) {
        const int from = (lk & 127) * 8;  // 16-byte pieces of the 128-byte rows of one channel half
        uint8_t* t = sv_ring + (ragged % VS) * TILE;
        for (int c = 0; c < HALVES; ++c)
          for (int x = from + lane; x < 1024; x += 32)
            *reinterpret_cast<uint4*>(t + c * 16384 + x * 16) = make_uint4(0u, 0u, 0u, 0u);
        umma_fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[ragged % VS]);
      }
    }
  } else if (warp >= 4) {
    const int i = (warp >> 2) - 1, r = tid & 127, ni = i ? n1 : n0;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
    const uint32_t s_addr = lane_addr + i * 128, o_addr = lane_addr + 256 + i * 128;
    const int rt = r / p.G, t = t0 + i * p.tokens + rt;
    const bool row_ok = rt < p.tokens && t < lq;
    const int klim = !row_ok ? 0 : p.causal ? max(0, min(lk, t + shift + 1)) : lk;  // keys this row reads
    const float sl = p.scale_log2;
    const uint64_t sl2 = pack_f2(sl, sl);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < ni; ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&s_full[i], static_cast<uint32_t>(j & 1)))) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t sv[4][32];
#pragma unroll
      for (int q = 0; q < 4; ++q) tmem_ld32(s_addr + q * 32, sv[q]);
      tmem_wait_ld();
      const int lim = klim - (j0 + j) * 128;
      if (!__all_sync(0xffffffffu, lim >= 128)) {
#pragma unroll
        for (int c = 0; c < 128; ++c)
          if (c >= lim) sv[c >> 5][c & 31] = 0xff800000u;  // -inf
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 128; c += 2)
        mx4[(c >> 1) & 3] = fmaxf(fmaxf(mx4[(c >> 1) & 3], __uint_as_float(sv[c >> 5][c & 31])),
                                  __uint_as_float(sv[c >> 5][(c & 31) + 1]));
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sl;
      const bool grow = mx > m + 8.f;
      if (__any_sync(0xffffffffu, grow)) {
        const float alpha = grow ? (m == -INFINITY ? 0.f : ex2_approx(m - mx)) : 1.f;
        if (j > 0) {  // O holds the tiles before this one once their P V is done
          if (!__all_sync(0xffffffffu, mbar_wait_bounded(&pv_done[i], static_cast<uint32_t>((j - 1) & 1)))) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t ov[32];
            tmem_ld32(o_addr + c * 32, ov);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
            tmem_st32(o_addr + c * 32, ov);
          }
          tmem_wait_st();
        }
        l *= alpha;
        if (grow) m = mx;
      }
      const float neg = m == -INFINITY ? 0.f : -m;  // nothing read yet: every score is -inf, P = 0
      const uint64_t neg2 = pack_f2(neg, neg);
      uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t pk[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const int c = h * 64 + 2 * e;
          const float2 x = unpack_f2(fma_f2(
              pack_f2(__uint_as_float(sv[c >> 5][c & 31]), __uint_as_float(sv[c >> 5][(c & 31) + 1])), sl2, neg2));
          const float a = ex2_approx(x.x), b = ex2_approx(x.y);
          pk[e] = M::pack(a, b);
          sum[e & 3] = add_f2(sum[e & 3], pack_f2(a, b));
        }
        tmem_st32(s_addr + h * 32, pk);
      }
      const float2 ts = unpack_f2(add_f2(add_f2(sum[0], sum[1]), add_f2(sum[2], sum[3])));
      l += ts.x + ts.y;
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[i]);
    }
    if (ok && ni > 0)
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&pv_done[i], static_cast<uint32_t>((ni - 1) & 1)));
    if (!ok) {
      report(p.status, LINATTN_DEV_TIMEOUT);
      dead = 1;
    }
    tc_fence_after();
    const float inv = l != 0.f ? 1.f / l : 0.f;
    const float lse = l != 0.f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
    const int64_t row = (static_cast<int64_t>(q_first) + t) * p.Hq + kvh * p.G + (r - rt * p.G);
    const bool have = ok && ni > 0;  // warp-uniform
    if (p.n_splits > 1) {
      if (row_ok) p.part_lse[blockIdx.y * (p.Nq * p.Hq) + row] = lse;
#pragma unroll 1
      for (int c = 0; c < (have ? D / 32 : 0); ++c) {
        uint32_t ov[32];
        tmem_ld32(o_addr + c * 32, ov);
        tmem_wait_ld();
        if (row_ok) {
          float4* dst = reinterpret_cast<float4*>(p.part_o + (blockIdx.y * (p.Nq * p.Hq) + row) * D + c * 32);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dst[e] = make_float4(__uint_as_float(ov[4 * e]) * inv, __uint_as_float(ov[4 * e + 1]) * inv,
                                 __uint_as_float(ov[4 * e + 2]) * inv, __uint_as_float(ov[4 * e + 3]) * inv);
        }
      }
    } else {
      if (row_ok && p.lse) p.lse[row] = lse;
      // rows staged in this row tile's Q (every MMA that reads it is done), then written
      // whole rows at a time: only the rows of this sequence
      uint8_t* st = sq + i * TILE;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t ov[32];
        if (have) {
          tmem_ld32(o_addr + c * 32, ov);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) ov[e] = 0u;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = l != 0.f ? M::pack(__uint_as_float(ov[q * 8 + 2 * e]) * inv, __uint_as_float(ov[q * 8 + 2 * e + 1]) * inv) : 0u;
          const int piece = (c & 1) * 4 + q;
          *reinterpret_cast<uint4*>(st + (c >> 1) * 16384 + r * 128 + ((piece ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      __syncwarp();
      constexpr int PIECES = D / 8, RPI = 32 / PIECES;  // 16-byte pieces of a row, rows of one step
      const int piece = lane % PIECES;
#pragma unroll 4
      for (int x = 0; x < 32; x += RPI) {
        const int rr = 32 * (warp & 3) + x + lane / PIECES, tt = rr / p.G, tok = t0 + i * p.tokens + tt;
        if (tt < p.tokens && tok < lq) {
          const uint4 w = *reinterpret_cast<const uint4*>(st + (piece >> 3) * 16384 + rr * 128 + (((piece & 7) ^ (rr & 7)) << 4));
          *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (static_cast<int64_t>(q_first) + tok) * p.ot +
                                    (static_cast<int64_t>(kvh) * p.G + rr - tt * p.G) * p.oh + piece * 8) = w;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (dead && tid == 32 && n > 0) {  // MMAs may still be in flight: wait for them before TMEM goes
    umma_commit(&last);
    (void)mbar_wait_bounded(&last, 0, 200000000ull);
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

int packed_fail(int code, const char* what) {
  char msg[256];
  snprintf(msg, sizeof(msg), "packed_attention: %s", what);
  return set_error(code, msg);
}

template <typename T, int D>
cudaError_t launch_packed(const PackedArgs& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, dim3 grid,
                          cudaStream_t st) {
  auto kern = packed_attention_kernel<T, D>;
  static int allowed[64] = {};
  const cudaError_t e = allow_smem(kern, PackedSmem<D>::BYTES, allowed);
  if (e != cudaSuccess) return e;
  kern<<<grid, PA_THREADS, PackedSmem<D>::BYTES, st>>>(p, q, k, v);
  return cudaGetLastError();
}

int64_t packed_tiles(int64_t N_q, int64_t G, int64_t S, int64_t max_q) {
  const int64_t rows = 2 * (128 / G);
  return lmin(N_q / rows + S, S * ((max_q + rows - 1) / rows));
}

}  // namespace

}  // namespace linattn

using namespace linattn;

extern "C" int32_t linattn_packed_attention_splits(int64_t N_q, int64_t Hq, int64_t Hkv, int64_t S, int64_t max_q,
                                                   int64_t max_k) {
  if (N_q < 1 || Hkv < 1 || Hq < Hkv || Hq / Hkv > 128 || S < 1 || max_q < 1) return 1;
  const int64_t ctas = packed_tiles(N_q, Hq / Hkv, S, max_q) * Hkv;
  // one wave of the GPU, with at least 4 key tiles to a part
  return static_cast<int32_t>(lmax(1, lmin(lmin(sm_count() / lmax(1, ctas), (max_k + 127) / 128 / 4), 32)));
}

extern "C" int64_t linattn_packed_attention_workspace(int64_t N_q, int64_t Hq, int64_t D, int32_t n_splits) {
  return n_splits > 1 ? static_cast<int64_t>(n_splits) * N_q * Hq * (D + 1) * 4 : 0;
}

extern "C" int linattn_packed_attention(const void* q, const void* k, const void* v, int32_t dtype, int64_t N_q, int64_t N_k,
                                        int64_t Hq, int64_t Hkv, int64_t D, const int64_t* q_strides,
                                        const int64_t* k_strides, const int64_t* v_strides, const int32_t* cu_q,
                                        const int32_t* cu_k, int64_t S, int64_t max_q, int64_t max_k, int32_t causal,
                                        float scale, void* out, const int64_t* out_strides, float* lse, int32_t n_splits,
                                        void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  if (!q_strides || !k_strides || !v_strides || !out_strides || !cu_q || !cu_k) return packed_fail(LINATTN_EINVAL, "NULL pointer");
  if (dtype != LINATTN_BF16 && dtype != LINATTN_F16) return packed_fail(LINATTN_EUNSUPPORTED, "q, k and v must be bf16 or f16");
  if (D != 64 && D != 128) return packed_fail(LINATTN_EUNSUPPORTED, "head_dim must be 64 or 128");
  if (Hkv < 1 || Hq < 1 || Hq % Hkv) return packed_fail(LINATTN_EINVAL, "H_q must be a multiple of H_kv");
  if (Hq / Hkv > 128) return packed_fail(LINATTN_EUNSUPPORTED, "at most 128 query heads to a kv head");
  if (N_q < 0 || N_k < 0 || S < 0 || max_q < 0 || max_k < 0 || n_splits < 1)
    return packed_fail(LINATTN_EINVAL, "sizes must not be negative");
  if (N_q >= (int64_t(1) << 30) || N_k >= (int64_t(1) << 30)) return packed_fail(LINATTN_EUNSUPPORTED, "at most 2^30 rows");
  if (!(scale > 0.f) || scale > 1e30f) return packed_fail(LINATTN_EINVAL, "scale must be positive and finite");
  if (N_q == 0 || S == 0) return LINATTN_OK;
  if (!q || !out || (N_k > 0 && (!k || !v))) return packed_fail(LINATTN_EINVAL, "NULL pointer");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
       reinterpret_cast<uintptr_t>(out)) % 16)
    return packed_fail(LINATTN_EINVAL, "q, k, v and out must be 16-byte aligned");
  for (int i = 0; i < 2; ++i)
    if (q_strides[i] % 8 || k_strides[i] % 8 || v_strides[i] % 8 || out_strides[i] % 8)
      return packed_fail(LINATTN_EINVAL, "strides must be multiples of 16 bytes");
  if (n_splits > 1 && (!workspace || workspace_bytes < linattn_packed_attention_workspace(N_q, Hq, D, n_splits) ||
                       reinterpret_cast<uintptr_t>(workspace) % 16))
    return packed_fail(LINATTN_EINVAL, "workspace too small or not 16-byte aligned");
  PackedArgs p;
  p.G = static_cast<int>(Hq / Hkv);
  p.tokens = 128 / p.G;
  const CUtensorMapDataType cu = dtype == LINATTN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap tq, tk, tv;
  const int64_t qd[3] = {D, Hq, N_q}, qs[2] = {q_strides[1] * 2, q_strides[0] * 2};
  const int64_t kd[3] = {D, Hkv, lmax(N_k, 1)}, ks[2] = {k_strides[1] * 2, k_strides[0] * 2}, vs[2] = {v_strides[1] * 2, v_strides[0] * 2};
  const int qbox[3] = {64, p.G, p.tokens}, kbox[3] = {64, 1, 128};
  const bool keys = N_k > 0;  // without keys no tile is read
  if (!tensor_map_3d(&tq, q, cu, qd, qs, qbox) || !tensor_map_3d(&tk, keys ? k : q, cu, kd, ks, kbox) ||
      !tensor_map_3d(&tv, keys ? v : q, cu, kd, vs, kbox))
    return packed_fail(LINATTN_ECUDA, "tensor map encoding failed");
  p.cu_q = cu_q; p.cu_k = cu_k; p.Nq = N_q; p.Nk = N_k;
  p.S = static_cast<int>(S); p.Hq = static_cast<int>(Hq); p.Hkv = static_cast<int>(Hkv);
  p.causal = causal ? 1 : 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = out; p.ot = out_strides[0]; p.oh = out_strides[1];
  p.lse = lse;
  p.n_splits = n_splits;
  p.part_o = static_cast<float*>(workspace);
  p.part_lse = n_splits > 1 ? p.part_o + n_splits * N_q * Hq * D : nullptr;
  p.status = status;
  const int64_t tiles = packed_tiles(N_q, p.G, S, max_q);
  if (tiles * Hkv >= (int64_t(1) << 31) || n_splits > 1024) return packed_fail(LINATTN_EUNSUPPORTED, "too many tiles");
  if (tiles == 0) return LINATTN_OK;
  const dim3 grid(static_cast<unsigned>(tiles * Hkv), static_cast<unsigned>(n_splits));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == LINATTN_BF16) e = D == 128 ? launch_packed<__nv_bfloat16, 128>(p, tq, tk, tv, grid, st) : launch_packed<__nv_bfloat16, 64>(p, tq, tk, tv, grid, st);
  else e = D == 128 ? launch_packed<__half, 128>(p, tq, tk, tv, grid, st) : launch_packed<__half, 64>(p, tq, tk, tv, grid, st);
  if (e == cudaSuccess && n_splits > 1) {
    // rows (token, head): the merge's innermost index is the head
    const int64_t os[4] = {0, out_strides[0], out_strides[1], 1};
    e = launch_lse_combine(p.part_o, p.part_lse, n_splits, N_q * Hq, D, out, dtype, N_q, Hq, os, lse, st);
  }
  return e == cudaSuccess ? LINATTN_OK : packed_fail(LINATTN_ECUDA, cudaGetErrorString(e));
}
