// Attention weight that each key of packed prompts has received:
//   mass[h, j] = sum over queries i that read j, heads g of kv head h, of 2^(c2 q_ig . k_j - lse2_ig)
// (c2 and lse2 in log2 units) on the 5th-generation tensor cores.
//
// The weights need each row's final lse, so this is a second pass over Q K^T, without V.
// The product is taken transposed, S^T = K Q^T: 128 keys of one kv head are the rows
// (TMEM lanes), so that a key's sum stays in one thread's registers over the whole pass:
// no reduction across threads, no atomics, a fixed order.  The columns are 128 / G tokens
// times the group's G heads, which one 3-D tensor-map box brings in as 128 rows.
//
// One CTA = 512 keys, four tiles of 128 that share every Q tile; warp 0 loads K once and Q
// tiles through a ring (TMA), warp 1 issues tcgen05.mma, a tile of keys to each of four TMEM
// buffers of 128 columns, and each buffer has a warpgroup: a thread reads its key's 128 scores,
// then one packed FMA, two exponentials and one packed add for two of them.  (Two warpgroups
// with a whole tile in registers left the pipes idle, 1570 us where four took 1290; with one
// key tile to a CTA and its Q tiles dealt to the warpgroups, a short window paid a CTA's start
// and end for every 128 keys.  CTAs that stay for the whole call, as the attention's, were 5% to
// 20% slower: the schedule is then fixed, and the next keys wait for the last product.)  Keys
// with the most queries (the first of a sequence) come first in the grid.
// Bound: the exponentials (16 a clock and SM: 1024 clocks a tile, against 512 for its MMAs
// at D = 128), 3 of 8 of which go to the FMA pipe instead.  Measured (32 / 8 heads, D = 128, bf16):
// 4096 tokens 92 us, 16384 tokens 1140 to 1290 us (850 to 960 TFLOP/s); FMA pipe 64%, exponential
// unit 57% busy.
#include <cstdio>
#include <type_traits>

#include "launchers.cuh"
#include "packed_tiles.cuh"
#include "umma.cuh"

namespace linattn {

namespace {

struct MassArgs {
  const float* lse;        // (N_q, H_q)
  const int32_t* cu_q;
  const int32_t* cu_k;
  int64_t Nq, Nk;
  int max_k;                  // keys of a sequence at most: later ones are not written
  int S, Hq, Hkv, G, tokens;  // tokens of a 128-row query tile (floor(128 / G))
  int causal;
  int64_t window;
  float scale_log2;
  float* mass;             // (n_splits, H_kv, N_k) with row stride mass_stride
  int64_t mass_stride, split_stride;
  int n_splits;
  int32_t* status;
};

constexpr int MT_GROUPS = 4;  // warpgroups on scores, each with a TMEM buffer of 128 columns
constexpr int MT_THREADS = 128 * (1 + MT_GROUPS);
constexpr int MT_KEYS = 128 * MT_GROUPS;  // keys of a CTA

// Of every 8 pairs of weights, those computed on the FMA pipe (ex2_poly2: up to 2.7e-6 off each, which
// a key that few queries read keeps; sums of thousands of them are 2.3e-7 off, 4.4e-8 with every
// weight and sum in fp32): none / 2 / 3 / 4 of 8 took 1379 / 1237 / 1210 / about 1400 us for 16384
// tokens, 32 / 8 heads, D = 128.
constexpr uint32_t MT_POLY = 0x52;


__device__ __forceinline__ uint64_t ex2_pair(uint64_t x) {
  const float2 v = unpack_f2(x);
  return pack_f2(ex2_approx(v.x), ex2_approx(v.y));
}

template <int D>
struct MassSmem {
  static constexpr int TILE = 128 * D * 2;
  static constexpr int STAGES = D == 128 ? 2 : 6;
  static constexpr int BYTES = 1024 + TILE * (MT_GROUPS + STAGES);
};

template <typename T, int D>
__global__ void __launch_bounds__(MT_THREADS, 1)
    attention_mass_kernel(const MassArgs p, const __grid_constant__ CUtensorMap tmq,
                          const __grid_constant__ CUtensorMap tmk) {
  using SM = MassSmem<D>;
  constexpr int ST = SM::STAGES, HALVES = D / 64;
  constexpr uint32_t IDESC = umma_idesc(std::is_same<T, __nv_bfloat16>::value ? 1 : 0, 128, 128, 0);
  extern __shared__ __align__(128) uint8_t msmem_raw[];
  uint8_t* sk = msmem_raw + ((1024 - (smem_u32(msmem_raw) & 1023)) & 1023);
  uint8_t* sq = sk + MT_GROUPS * SM::TILE;
  __shared__ __align__(8) uint64_t k_full[MT_GROUPS], q_full[ST], q_empty[ST], s_full[MT_GROUPS], s_empty[MT_GROUPS], last;
  __shared__ uint32_t tmem_sh;
  __shared__ int dead;
  __shared__ __align__(16) float nl[MT_GROUPS][2][128];  // [warpgroup][parity][column]: -lse2, or -inf for a column that does not count

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // the parts of the keys with the most queries come first
  const int split = blockIdx.x % p.n_splits, kvh = blockIdx.x / p.n_splits % p.Hkv;
  PackedTile tl;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!packed_tile(p.cu_k, p.cu_q, p.S, p.Nk, p.Nq, MT_KEYS, p.max_k, blockIdx.x / p.n_splits / p.Hkv, &tl)) return;
  if (!tl.sound && tid == 0) report(p.status, LINATTN_DEV_BAD_ID);
  const int k_first = tl.first, lk = tl.n, q_first = tl.other_first, lq = tl.other_n;
  const int key0 = tl.tile * MT_KEYS, shift = lk - lq;  // query i stands at position i + shift
  const int keys = min(lk, p.max_k);
  const int key_tiles = min(MT_GROUPS, (keys - key0 + 127) >> 7);
  // query tiles that read these keys, and this split's share of them
  const int w_lo = p.window > 0 && p.window < lq ? lq - static_cast<int>(p.window) : 0;
  const int q_lo = max(w_lo, p.causal ? key0 - shift : 0);
  int qt0 = q_lo / p.tokens;
  int n = max(0, (lq + p.tokens - 1) / p.tokens - qt0);
  if (q_lo >= lq) n = 0;
  if (p.n_splits > 1) {
    const int share = (n + p.n_splits - 1) / p.n_splits, at = min(n, split * share);
    qt0 += at;
    n = min(n - at, share);
  }
  // the first of these tiles that key tile x takes part in (a later key has fewer queries)
  auto begins = [&](int x) {
    const int first = max(w_lo, p.causal ? key0 + 128 * x - shift : 0);
    return x < key_tiles && first < lq ? max(0, first / p.tokens - qt0) : n;
  };
  const int boxb = p.tokens * p.G * 128;  // bytes of one 64-channel box of queries

  if (tid == 0) {
    mbar_init(&last, 1);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
    }
    for (int s = 0; s < MT_GROUPS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&s_empty[s], 128);
    }
    dead = 0;
    mbar_fence_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_sh)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // rows of a query tile that no box ever fills (128 is no multiple of G)
  const int idle = 128 - p.tokens * p.G;
  for (int i = tid; i < ST * HALVES * idle * 8; i += MT_THREADS) {
    const int box = i / (idle * 8), at = i - box * (idle * 8);
    *reinterpret_cast<uint4*>(sq + (box / HALVES) * SM::TILE + (box % HALVES) * 16384 + boxb + at * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  umma_fence_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_sh;

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      // a key tile that none of these queries reads is not loaded: nothing would wait for it
      auto load_k = [&](int x) {
        if (begins(x) >= n) return;
        mbar_arrive_expect_tx(&k_full[x], SM::TILE);
        for (int c = 0; c < HALVES; ++c)
          tma_load_3d(sk + x * SM::TILE + c * 16384, &tmk, 64 * c, kvh, k_first + key0 + 128 * x, &k_full[x]);
      };
      load_k(0);
      int issued = 0;
      for (int j = 0; j < n; ++j) {
        const int st = j % ST;
        if (j >= ST && !mbar_wait_bounded(&q_empty[st], static_cast<uint32_t>((j / ST - 1) & 1))) {
          report(p.status, LINATTN_DEV_TIMEOUT);
          dead = 1;
          break;
        }
        if (dead) break;
        mbar_arrive_expect_tx(&q_full[st], boxb * HALVES);
        for (int c = 0; c < HALVES; ++c)
          tma_load_3d(sq + st * SM::TILE + c * 16384, &tmq, 64 * c, kvh * p.G, q_first + (qt0 + j) * p.tokens, &q_full[st]);
        issued = j + 1;
        if (j == 0)
          for (int x = 1; x < key_tiles; ++x) load_k(x);
      }
      if (dead) {  // the copies in flight land before the CTA gives up its shared memory
        for (int x = 0; x < (issued > 0 ? key_tiles : 1); ++x)
          if (begins(x) < n) (void)mbar_wait_bounded(&k_full[x], 0, 200000000ull);
        for (int j = issued > ST ? issued - ST : 0; j < issued; ++j)
          (void)mbar_wait_bounded(&q_full[j % ST], static_cast<uint32_t>((j / ST) & 1), 200000000ull);
      }
    }
  } else if (warp == 1) {
    if (n > 0) {
      bool ok = true;
      const uint64_t k_desc = umma_desc(smem_u32(sk), 16, 1024), q_desc = umma_desc(smem_u32(sq), 16, 1024);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      int from[MT_GROUPS];
#pragma unroll
      for (int x = 0; x < MT_GROUPS; ++x) from[x] = begins(x);
      for (int j = 0; ok && j < n; ++j) {
        const int st = j % ST;
        ok = warp_wait(&q_full[st], static_cast<uint32_t>((j / ST) & 1));
        const uint64_t qd = q_desc + st * (SM::TILE >> 4);
#pragma unroll
        for (int x = 0; x < MT_GROUPS; ++x) {
          if (!ok || j < from[x]) continue;
          const int round = j - from[x];  // of this buffer
          if (round == 0) ok = warp_wait(&k_full[x], 0);
          else ok = warp_wait(&s_empty[x], static_cast<uint32_t>((round - 1) & 1));
          if (!ok) break;
          tc_fence_after();
          if (elect_lane()) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t off = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
              umma_f16(tm + x * 128, k_desc + x * (SM::TILE >> 4) + off, qd + off, IDESC, kk > 0 ? 1u : 0u);
            }
            umma_commit(&s_full[x]);
          }
        }
        if (ok && elect_lane()) umma_commit(&q_empty[st]);
      }
      if (!ok && lane == 0) {
        report(p.status, LINATTN_DEV_TIMEOUT);
        dead = 1;
      }
    }
  } else if (warp >= 4) {
    const int wg = (warp >> 2) - 1, c = tid & 127;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
    const int tile0 = key0 + 128 * wg, key = tile0 + c;  // this warpgroup's keys, this thread's
    const int ct = c / p.G, cg = c - ct * p.G;
    const bool used = ct < p.tokens;
    // -lse2 of column c of tile j
    auto column = [&](int j) -> float {
      const int i = (qt0 + j) * p.tokens + ct;
      if (j >= n || !used || i >= lq || i < w_lo) return -INFINITY;
      const float l = p.lse[(static_cast<int64_t>(q_first) + i) * p.Hq + kvh * p.G + cg];
      return l == -INFINITY ? -INFINITY : -l * 1.4426950408889634f;
    };
    const uint64_t c2 = pack_f2(p.scale_log2, p.scale_log2);
    float total = 0.f;
    bool ok = true;
    const int from = begins(wg);
    float mine = column(from);
    for (int j = from; j < n; ++j) {
      const int par = (j - from) & 1;
      float* row = nl[wg][par];
      row[c] = mine;
      // every column with a query counts for every key of the tile (the rows of a tile that
      // hold none are zeros, and their -inf leaves nothing of them)
      const int pos0 = (qt0 + j) * p.tokens + shift;
      int whole = (((mine == mine && mine != -INFINITY) || !used) && (!p.causal || pos0 >= tile0 + 127)) ? 1 : 0;
      asm volatile(
          "{\n\t.reg .pred a, b;\n\tsetp.ne.s32 a, %0, 0;\n\t"
          "barrier.cta.red.and.pred b, %1, 128, a;\n\tselp.s32 %0, 1, 0, b;\n\t}"
          : "+r"(whole)
          : "r"(1 + wg)
          : "memory");
      mine = column(j + 1);
      // a warp whose wait gave up goes on through the named barriers, without scores
      ok = ok && warp_wait(&s_full[wg], static_cast<uint32_t>(par));
      if (!ok) continue;
      tc_fence_after();
      // columns of queries before this key, past the sequence or outside the window do not
      // count, whatever their scores are
      const int c_lo = p.causal ? max(0, key - pos0) * p.G : 0;
      uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t sv[32];
        tmem_ld32(lane_addr + wg * 128 + q * 32, sv);
        tmem_wait_ld();
        if (q == 3) {
          tc_fence_before();
          mbar_arrive(&s_empty[wg]);
        }
        if (whole) {  // MT_POLY of every 8 pairs of weights on the FMA pipe
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 b = *reinterpret_cast<const float4*>(row + q * 32 + e * 4);
            const uint64_t x = fma_f2(pack_f2(__uint_as_float(sv[4 * e]), __uint_as_float(sv[4 * e + 1])), c2, pack_f2(b.x, b.y));
            const uint64_t y = fma_f2(pack_f2(__uint_as_float(sv[4 * e + 2]), __uint_as_float(sv[4 * e + 3])), c2, pack_f2(b.z, b.w));
            sum[e & 1] = add_f2(sum[e & 1], ((MT_POLY >> ((2 * e) & 7)) & 1) ? ex2_poly2(x) : ex2_pair(x));
            sum[2 + (e & 1)] = add_f2(sum[2 + (e & 1)], ((MT_POLY >> ((2 * e + 1) & 7)) & 1) ? ex2_poly2(y) : ex2_pair(y));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float b0 = row[q * 32 + e], b1 = row[q * 32 + e + 1];
            const bool in0 = q * 32 + e >= c_lo && b0 != -INFINITY, in1 = q * 32 + e + 1 >= c_lo && b1 != -INFINITY;
            const float x0 = fmaf(__uint_as_float(sv[e]), p.scale_log2, b0), x1 = fmaf(__uint_as_float(sv[e + 1]), p.scale_log2, b1);
            sum[(e >> 1) & 3] = add_f2(sum[(e >> 1) & 3], pack_f2(in0 ? ex2_approx(x0) : 0.f, in1 ? ex2_approx(x1) : 0.f));
          }
        }
      }
      const float2 t = unpack_f2(add_f2(add_f2(sum[0], sum[1]), add_f2(sum[2], sum[3])));
      total += t.x + t.y;
    }
    if (!ok) {
      report(p.status, LINATTN_DEV_TIMEOUT);
      dead = 1;
    }
    if (key < keys) p.mass[split * p.split_stride + kvh * p.mass_stride + k_first + key] = total;
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

// mass = sum of the splits' parts, in their order.  Keys that the parts do not cover (no
// sequence's) are left alone.
__global__ void __launch_bounds__(256) mass_sum_kernel(const float* __restrict__ parts, int n_splits, int64_t split_stride,
                                                       int64_t Nk, const int32_t* cu, int S, int max_k,
                                                       float* __restrict__ mass, int64_t mass_stride) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  PackedOwner owner;
  owner.load(cu, S, Nk, max_k);
  const float* p = parts + blockIdx.y * Nk + lmin(j, Nk - 1);
  float s = 0.f;
#pragma unroll 8
  for (int i = 0; i < n_splits; ++i) s += p[i * split_stride];
  if (owner.has(j) && j < Nk) mass[blockIdx.y * mass_stride + j] = s;
}

int mass_fail(int code, const char* what) {
  char msg[256];
  snprintf(msg, sizeof(msg), "attention_mass: %s", what);
  return set_error(code, msg);
}

template <typename T, int D>
cudaError_t launch_mass(const MassArgs& p, const CUtensorMap& q, const CUtensorMap& k, unsigned grid, cudaStream_t st) {
  auto kern = attention_mass_kernel<T, D>;
  static int allowed[64] = {};
  const cudaError_t e = allow_smem(kern, MassSmem<D>::BYTES, allowed);
  if (e != cudaSuccess) return e;
  return launch_ahead(kern, dim3(grid), MT_THREADS, MassSmem<D>::BYTES, st, p, q, k);
}

}  // namespace

}  // namespace linattn

using namespace linattn;

extern "C" int32_t linattn_attention_mass_splits(int64_t Hq, int64_t Hkv, int64_t S, int64_t max_q, int64_t max_k,
                                                 int64_t window) {
  if (Hkv < 1 || Hq < Hkv || S < 1 || max_q < 1 || max_k < 1) return 1;
  const int64_t tokens = lmax(1, 128 / (Hq / Hkv));
  // all but the longest sequence are taken to be half as long
  const int64_t ctas = (((S + 1) * ((max_k + MT_KEYS - 1) / MT_KEYS) + 1) / 2) * Hkv;
  const int64_t q_tiles = ((window > 0 ? lmin(window, max_q) : max_q) + tokens - 1) / tokens;
  const int64_t sms = sm_count();
  // CTAs differ in length (causal), so a few rounds of the GPU: two where one split leaves SMs
  // idle, else three (4096 tokens, D = 128: 2 / 3 / 4 / 6 rounds 91 / 92 / 96 / 103 us; 8192
  // tokens, D = 64: 315 / 299 / 301 / 304).  At least 2 query tiles to a split.  Measured in us,
  // by splits:
  //   a prompt of 1500 tokens, 8 kv heads of 32: 1: 105, 5: 32, 8: 25, 12: 27, 16: 29
  //   ten prompts of 5 to 923 tokens, 2 kv heads of 8: 1: 63, 3: 30, 6: 20, 8: 18, 12: 19
  //   prompts of 385 and 232 tokens, 4 kv heads of 20: 1: 33, 4: 16, 8: 12, 16: 11
  // Few query tiles do not pay for the second launch (8 prompts of up to 128 tokens, 4 tiles: 10.9
  // us and 10.5 with 2 splits, 18.5 and 26.9 with the host's call; 8 tiles: 16.9 and 10.8 with 4).
  if (ctas >= 3 * sms || q_tiles < 6) return 1;
  const int64_t rounds = ctas < sms ? 2 : 3;
  return static_cast<int32_t>(lmax(1, lmin(lmin((rounds * sms + ctas - 1) / ctas, q_tiles / 2), 64)));
}

extern "C" int64_t linattn_attention_mass_workspace(int64_t N_k, int64_t Hkv, int32_t n_splits) {
  return n_splits > 1 ? static_cast<int64_t>(n_splits) * N_k * Hkv * 4 : 0;
}

extern "C" int linattn_attention_mass(const void* q, const void* k, int32_t dtype, int64_t N_q, int64_t N_k, int64_t Hq,
                                      int64_t Hkv, int64_t D, const int64_t* q_strides, const int64_t* k_strides,
                                      const float* lse, const int32_t* cu_q, const int32_t* cu_k, int64_t S,
                                      int64_t max_q, int64_t max_k, int32_t causal, int64_t window, float scale,
                                      float* mass, int64_t mass_stride, int32_t n_splits, void* workspace,
                                      int64_t workspace_bytes, int32_t* status, void* stream) {
  if (!q_strides || !k_strides || !cu_q || !cu_k) return mass_fail(LINATTN_EINVAL, "NULL pointer");
  if (dtype != LINATTN_BF16 && dtype != LINATTN_F16) return mass_fail(LINATTN_EUNSUPPORTED, "q and k must be bf16 or f16");
  if (D != 64 && D != 128) return mass_fail(LINATTN_EUNSUPPORTED, "head_dim must be 64 or 128");
  if (Hkv < 1 || Hq < 1 || Hq % Hkv) return mass_fail(LINATTN_EINVAL, "H_q must be a multiple of H_kv");
  if (Hq / Hkv > 128) return mass_fail(LINATTN_EUNSUPPORTED, "at most 128 query heads to a kv head");
  if (N_q < 0 || N_k < 0 || S < 0 || max_q < 0 || max_k < 0 || window < 0 || n_splits < 1)
    return mass_fail(LINATTN_EINVAL, "sizes must not be negative");
  if (N_q >= (int64_t(1) << 30) || N_k >= (int64_t(1) << 30)) return mass_fail(LINATTN_EUNSUPPORTED, "at most 2^30 rows");
  if (!(scale > 0.f) || scale > 1e30f) return mass_fail(LINATTN_EINVAL, "scale must be positive and finite");
  if (N_k == 0 || S == 0) return LINATTN_OK;
  if (!k || !mass || (N_q > 0 && (!q || !lse))) return mass_fail(LINATTN_EINVAL, "NULL pointer");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k)) % 16 || q_strides[0] % 8 || q_strides[1] % 8 ||
      k_strides[0] % 8 || k_strides[1] % 8)
    return mass_fail(LINATTN_EINVAL, "q and k rows must be 16-byte aligned");
  if (n_splits > 1 && (!workspace || workspace_bytes < linattn_attention_mass_workspace(N_k, Hkv, n_splits)))
    return mass_fail(LINATTN_EINVAL, "workspace too small");
  const CUtensorMapDataType cu = dtype == LINATTN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  MassArgs p;
  p.G = static_cast<int>(Hq / Hkv);
  p.tokens = 128 / p.G;
  CUtensorMap tq, tk;
  const int64_t kd[3] = {D, Hkv, N_k}, ks[2] = {k_strides[1] * 2, k_strides[0] * 2};
  const int kbox[3] = {64, 1, 128};
  const int64_t qd[3] = {D, Hq, lmax(N_q, 1)}, qs[2] = {q_strides[1] * 2, q_strides[0] * 2};
  const int qbox[3] = {64, p.G, p.tokens};
  if (!tensor_map_3d(&tk, k, cu, kd, ks, kbox) || !tensor_map_3d(&tq, N_q > 0 ? q : k, cu, qd, qs, qbox))
    return mass_fail(LINATTN_ECUDA, "tensor map encoding failed");
  p.lse = lse; p.cu_q = cu_q; p.cu_k = cu_k; p.Nq = N_q; p.Nk = N_k;
  p.max_k = static_cast<int>(lmin(max_k, N_k));
  p.S = static_cast<int>(S); p.Hq = static_cast<int>(Hq); p.Hkv = static_cast<int>(Hkv);
  p.causal = causal ? 1 : 0;
  p.window = window;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.mass = n_splits > 1 ? static_cast<float*>(workspace) : mass;
  p.mass_stride = n_splits > 1 ? N_k : mass_stride;
  p.split_stride = n_splits > 1 ? N_k * Hkv : 0;
  p.n_splits = n_splits;
  p.status = status;
  const int64_t tiles = lmin(N_k / MT_KEYS + S, S * ((max_k + MT_KEYS - 1) / MT_KEYS));
  if (n_splits > 65535 || tiles * Hkv * n_splits >= (int64_t(1) << 31)) return mass_fail(LINATTN_EUNSUPPORTED, "too many tiles");
  if (tiles == 0) return LINATTN_OK;
  const unsigned grid = static_cast<unsigned>(tiles * Hkv * n_splits);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == LINATTN_BF16) e = D == 128 ? launch_mass<__nv_bfloat16, 128>(p, tq, tk, grid, st) : launch_mass<__nv_bfloat16, 64>(p, tq, tk, grid, st);
  else e = D == 128 ? launch_mass<__half, 128>(p, tq, tk, grid, st) : launch_mass<__half, 64>(p, tq, tk, grid, st);
  if (e == cudaSuccess && n_splits > 1) {
    e = launch_ahead(mass_sum_kernel, dim3(static_cast<unsigned>((N_k + 255) / 256), static_cast<unsigned>(Hkv)), 256, 0, st,
                     static_cast<const float*>(workspace), static_cast<int>(n_splits), static_cast<int64_t>(p.split_stride), N_k, cu_k,
                     p.S, p.max_k, mass, mass_stride);
  }
  return e == cudaSuccess ? LINATTN_OK : mass_fail(LINATTN_ECUDA, cudaGetErrorString(e));
}
