// One query token per sequence over the slots of the heavy-hitter cache, with the weights
// added to the slots' masses.
//
//   o = sum_n p_n v_n,  p_n = exp(c q . k_n - lse),  mass_n += sum over the group's heads of p_n
//
// HBM-bound: K and V are read once (2 D elements a slot), everything else is small.  One CTA to
// an SM stays for the whole call and takes an equal share of all 128-slot tiles of all
// (sequence, kv head) units, in order, so that no SM idles at the end whatever the lengths
// are; a producer warp keeps a ring of tiles (K and V, 128-byte-swizzled tensor-map boxes) full,
// across units too, so that the memory never waits for a unit's epilogue.  Eight warps work on
// a tile: for S^T = K Q^T (mma.sync, 8 heads as columns) a warp has 16 slots, the weights go
// through shared memory, and for O^T = V^T P^T a warp has 16 channels and all 128 slots (D = 64:
// half of them), so that o is not spread over warps; one barrier a tile.  P is split into
// hi + lo 16-bit parts (to ~2^-16), so o carries its own rounding only.
//
// The masses need a unit's final lse, so its scores are kept until then, and four more warps
// finish a unit while the others go on with the next one (done by the same warps, through global
// memory, the masses cost 59 of 205 us at 64 sequences x 8 heads x 4096 slots).  A unit that one
// CTA has whole keeps its scores in tensor memory, which this kernel has no other use for: a warp
// stores its accumulator fragments as they are, 4 columns a tile, and the finishing warp of the
// same 32 lanes reads them back (4096 slots a unit for up to 8 heads, twice over; through the
// workspace in global memory the call took 6 us more).  Longer ones, and units that
// several CTAs share, go through the workspace.  A shared unit's (o, m, l) are merged by the
// finishing warps of the last CTA to arrive at it: the parts are added in their order, whoever
// does it, so results do not depend on it.  When a CTA has no more tiles, its other eight warps
// help with its last unit.  Sequences x heads x slots in us, with the merge done by the warps that
// have the tiles / by the finishing warps (bf16, 4 query heads to a kv head):
//   1 x 8 x 2048, D = 128: 11.8 / 10.7     2 x 8 x 2048: 14.7 / 12.7     8 x 8 x 2048: 20.0 / 18.4
//   64 x 8 x 512: 37.8 / 33.9              12 x 8 x 4096: 44.8 / 47.0    64 x 8 x 4096: 157 / 156
//   24 x 8 x 1978, D = 64: 31.6 / 29.0     64 x 8 x 1978: 60.8 / 55.7
#include <cstdio>
#include <cstring>
#include <type_traits>

#include "launchers.cuh"
#include "sparse_attention_mma.cuh"
#include "umma.cuh"

namespace linattn {

namespace {

struct HeavyAttendArgs {
  float* mass;
  const int32_t* seen;
  const void* q;
  void* out;
  int64_t qb, qh, ob, oh;
  int B, H, M, G;
  int h0, heads;     // heads [h0, h0 + heads) of every group in this launch
  float scale_log2;
  int accumulate;
  int Ms;            // M up to a multiple of 4
  float* scores;     // (B * H, heads, Ms) log2-domain scores
  float* part_o;     // (CTAs, 2, HN, D) unnormalised o of units that this CTA shares
  float* part_ml;    // (CTAs, 2, 2, HN) their maxima and sums
  int32_t* ticket;   // (B * H) zeros: arrivals at a shared unit
  int32_t* status;
};

constexpr int AT_WARPS = 8;                     // on tiles; then one that loads, and the finishing warps
constexpr int AT_FINISH = 128;                  // threads that finish units
constexpr int AT_THREADS = 32 * (AT_WARPS + 1) + AT_FINISH;
constexpr int AT_ROWS = 128;                    // slots of a tile
constexpr int AT_BOX = 128;                     // slots of one tensor-map box
constexpr int AT_PROW = AT_ROWS * 2 + 16;       // bytes of a row of P: banks apart
constexpr int AT_PARTS = 160;                   // CTAs that may share a unit: more than the GPU has SMs

template <int D, int NT>
struct AttendSmem {
  static constexpr int HN = 8 * NT;
  static constexpr int HALF = AT_ROWS * 128;              // 64 channels of K or V
  static constexpr int STAGE = 2 * (D / 64) * HALF;       // K then V
  static constexpr int STAGES = D == 64 ? (NT == 4 ? 4 : 6) : NT == 4 ? 2 : 3;
  static constexpr int P = 2 * 2 * HN * AT_PROW;          // [buffer][hi, lo][head][slot]
  static constexpr int WEIGHTS = AT_PARTS * HN * 4;       // of the parts of a shared unit
  static constexpr int BYTES = 1024 + STAGES * STAGE + P + WEIGHTS;
};

// The units of one CTA's share of the tiles, in order.
struct AttendWalk {
  const int32_t* seen;
  int B, H, M;
  int b, h, count, tiles;  // the current unit
  __device__ __forceinline__ void sequence(int at) {
    b = at;
    count = b < B ? min(max(seen[b], 0), M) : 0;
    tiles = (count + AT_ROWS - 1) / AT_ROWS;
  }
  __device__ __forceinline__ void next() {
    if (++h < H) return;
    h = 0;
    do sequence(b + 1);
    while (b < B && tiles == 0);
  }
};

__device__ __forceinline__ bool attend_barrier_or(bool x) {
  int r = x ? 1 : 0;
  asm volatile(
      "{\n\t.reg .pred a, b;\n\tsetp.ne.s32 a, %0, 0;\n\t"
      "barrier.cta.red.or.pred b, 1, 256, a;\n\tselp.s32 %0, 1, 0, b;\n\t}"
      : "+r"(r)
      :
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const float (&v)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(__float_as_uint(v[0])),
               "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3]))
               : "memory");
}
// The finishing warps'.
__device__ __forceinline__ void finish_barrier() { asm volatile("barrier.cta.sync 3, 128;" ::: "memory"); }
__device__ __forceinline__ bool finish_barrier_and(bool x) {
  int r = x ? 1 : 0;
  asm volatile(
      "{\n\t.reg .pred a, b;\n\tsetp.ne.s32 a, %0, 0;\n\t"
      "barrier.cta.red.and.pred b, 3, 128, a;\n\tselp.s32 %0, 1, 0, b;\n\t}"
      : "+r"(r)
      :
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void attend_barrier() { asm volatile("barrier.cta.sync 1, 256;" ::: "memory"); }

template <typename T, int D, int NT>
__global__ void __launch_bounds__(AT_THREADS, 1)
    heavy_attend_kernel(const HeavyAttendArgs a, const __grid_constant__ CUtensorMap tmk,
                        const __grid_constant__ CUtensorMap tmv) {
  using M = MmaOp<T>;
  using SM = AttendSmem<D, NT>;
  constexpr int HN = SM::HN, ST = SM::STAGES, HALVES = D / 64, CT = D / 16;
  extern __shared__ __align__(128) uint8_t atsmem_raw[];
  uint8_t* ring = atsmem_raw + ((1024 - (smem_u32(atsmem_raw) & 1023)) & 1023);
  uint8_t* pbuf = ring + ST * SM::STAGE;
  float* weights_sh = reinterpret_cast<float*>(pbuf + SM::P);  // [part][head]
  __shared__ __align__(8) uint64_t full[ST], empty[ST], job_full[2], job_empty[2];
  __shared__ float mx_w[AT_WARPS][HN], l_w[AT_WARPS][HN];
  // units on their way to the finishing warps: maxima and reciprocal sums of the heads
  __shared__ float fin[2][2][HN];
  __shared__ int64_t job_unit[2];
  __shared__ int64_t job_out[2];  // of its outputs
  __shared__ int job_count[2];  // slots in use
  __shared__ int job_c0[2], job_parts[2];  // the CTAs that share it; 1: none, fin is set
  __shared__ int job_tmem[2];   // scores in tensor memory
  __shared__ int job_next[2];   // else: the slots / 4 that warps have taken
  __shared__ int job_last[2];   // the CTA's last unit: the tile warps take part
  __shared__ uint32_t tmem_sh;
  __shared__ float upper[D == 64 ? 4 * 32 * 4 * NT : 1];  // D = 64: o of the tile's upper slots
  __shared__ int dead, arrived, help;
  __shared__ int64_t share[3];  // first tile, end, all tiles
  __shared__ int start[2];      // first tile's sequence, and its tile among the sequence's

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], AT_WARPS);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&job_full[s], 1);
      mbar_init(&job_empty[s], AT_FINISH);
    }
    dead = 0;
    mbar_fence_init();
  }
  if (warp == AT_WARPS + 1 && a.accumulate) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_sh)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // this CTA's share of the tiles
  if (warp == 0) {
    auto tiles_of = [&](int b) {
      return b < a.B ? static_cast<int64_t>((min(max(a.seen[b], 0), a.M) + AT_ROWS - 1) / AT_ROWS) * a.H : int64_t(0);
    };
    const int64_t early = tiles_of(lane);  // of the first 32 sequences
    int64_t all = early;
    for (int b = lane + 32; b < a.B; b += 32) all += tiles_of(b);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    const int64_t ctas = lmin(gridDim.x, all), c = blockIdx.x;
    const int64_t lo = c < ctas ? c * all / ctas : 0, hi = c < ctas ? (c + 1) * all / ctas : 0;
    if (lane == 0) {
      share[0] = lo;
      share[1] = hi;
      share[2] = all;
    }
    if (hi > lo) {
      int64_t base = 0;
      for (int b0 = 0; b0 < a.B && base <= lo; b0 += 32) {
        const int64_t mine = b0 == 0 ? early : tiles_of(b0 + lane);
        int64_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        if (lo >= base + incl - mine && lo < base + incl) {
          start[0] = b0 + lane;
          start[1] = static_cast<int>(lo - (base + incl - mine));
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
      }
    }
  }
  __syncthreads();
  tc_fence_after();
  const int64_t t0 = share[0], t1 = share[1], total = share[2];
  const int64_t nc = lmin(gridDim.x, total);
  // sequences without slots: o = 0
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if (a.seen[b] <= 0)
      for (int i = tid; i < a.H * a.heads * D; i += AT_THREADS) {
        const int head = i / D;
        static_cast<T*>(a.out)[b * a.ob + (static_cast<int64_t>(head / a.heads) * a.G + a.h0 + head % a.heads) * a.oh + i % D] = T(0.f);
      }
  // tensor memory: two units' scores of 256 columns, of a unit 128 columns for each warp of a
  // lane quarter, 4 NT columns a tile
  const uint32_t tmem = a.accumulate ? tmem_sh : 0;
  auto free_tmem = [&] {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  };
  if (t1 <= t0) {
    if (warp == AT_WARPS + 1 && a.accumulate) free_tmem();
    return;
  }
  AttendWalk w{a.seen, a.B, a.H, a.M};
  w.sequence(start[0]);
  w.h = start[1] / w.tiles;
  int first = start[1] % w.tiles;  // of this CTA in its first unit

  if (warp == AT_WARPS) {
    if (lane == 0) {
      int j = 0;
      bool ok = true;
      for (int64_t t = t0; ok && t < t1;) {
        const int end = static_cast<int>(lmin(w.tiles, first + (t1 - t)));
        const int64_t row0 = (static_cast<int64_t>(w.b) * a.H + w.h) * a.M;
        for (int i = first; ok && i < end; ++i, ++j) {
          const int st = j % ST;
          if (j >= ST) ok = mbar_wait_bounded(&empty[st], static_cast<uint32_t>((j / ST - 1) & 1));
          if (!ok || dead) {
            ok = false;
            break;
          }
          uint8_t* dst = ring + st * SM::STAGE;
          const int boxes = (min(AT_ROWS, w.count - i * AT_ROWS) + AT_BOX - 1) / AT_BOX;
          const int y = static_cast<int>(row0 + static_cast<int64_t>(i) * AT_ROWS);
          mbar_arrive_expect_tx(&full[st], static_cast<uint32_t>(boxes) * 2 * HALVES * AT_BOX * 128);
          for (int x = 0; x < boxes; ++x)
#pragma unroll
            for (int c = 0; c < HALVES; ++c)
              tma_load_3d(dst + c * SM::HALF + x * AT_BOX * 128, &tmk, 64 * c, y + x * AT_BOX, 0, &full[st]);
          for (int x = 0; x < boxes; ++x)
#pragma unroll
            for (int c = 0; c < HALVES; ++c)
              tma_load_3d(dst + (HALVES + c) * SM::HALF + x * AT_BOX * 128, &tmv, 64 * c, y + x * AT_BOX, 0, &full[st]);
        }
        t += end - first;
        first = 0;
        w.next();
      }
      if (!ok) {
        report(a.status, LINATTN_DEV_TIMEOUT);
        dead = 1;
      }
      // the copies in flight land before the CTA gives up its shared memory
      for (int i = j > ST ? j - ST : 0; i < j; ++i)
        (void)mbar_wait_bounded(&full[i % ST], static_cast<uint32_t>((i / ST) & 1), 200000000ull);
    }
    return;
  }

  // A finished unit's weights into its masses, by four warps (group) of each of the groups.
  auto add_tmem = [&](int x, int64_t unit, int count, int group, int groups) {
    float* mass = a.mass + unit * a.M;
    // this lane's scores of a tile: slots g and g + 8 of the two warps of its quarter, heads
    // 2 tig and 2 tig + 1 (of every 8)
    const int g = lane >> 2, tig = lane & 3, quarter = warp & 3;
    float f0[NT][2], f1[NT][2];
#pragma unroll
    for (int y = 0; y < NT; ++y)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int head = y * 8 + 2 * tig + e;
        f0[y][e] = fin[x][0][head];
        f1[y][e] = head < a.heads ? fin[x][1][head] : 0.f;
      }
    constexpr int STEP = NT >= 4 ? 1 : 4 / NT;  // tiles of 16 columns
    constexpr int BATCH = 2 * STEP;             // tiles whose masses are fetched together
    const int tiles = (count + AT_ROWS - 1) / AT_ROWS;
    for (int i0 = group * BATCH; i0 < tiles; i0 += groups * BATCH) {
      // lane tig = 0 owns slot g, tig = 1 slot g + 8
      const int n0 = i0 * AT_ROWS + 16 * quarter + g + 8 * tig;
      float old[2][BATCH];
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < BATCH; ++e) {
          const int n = n0 + 64 * half + e * AT_ROWS;
          old[half][e] = tig < 2 && n < count ? mass[n] : 0.f;
        }
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int s0 = 0; s0 < BATCH; s0 += STEP) {
          if (i0 + s0 >= tiles) continue;
          uint32_t sv[16];
          tmem_ld16(tmem + (static_cast<uint32_t>(32 * quarter) << 16) + x * 256 + half * 128 + (i0 + s0) * 4 * NT, sv);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < STEP; ++e) {
            float lo = 0.f, hi = 0.f;
#pragma unroll
            for (int y = 0; y < NT; ++y)
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                lo += ex2_approx(__uint_as_float(sv[((e * NT + y) * 4 + z) & 15]) - f0[y][z]) * f1[y][z];
                hi += ex2_approx(__uint_as_float(sv[((e * NT + y) * 4 + 2 + z) & 15]) - f0[y][z]) * f1[y][z];
              }
            lo += __shfl_xor_sync(0xffffffffu, lo, 1);
            hi += __shfl_xor_sync(0xffffffffu, hi, 1);
            lo += __shfl_xor_sync(0xffffffffu, lo, 2);
            hi += __shfl_xor_sync(0xffffffffu, hi, 2);
            const int n = n0 + 64 * half + (s0 + e) * AT_ROWS;
            if (tig < 2 && n < count) mass[n] = old[half][s0 + e] + (tig == 0 ? lo : hi);
          }
        }
    }
  };
  // The same from the workspace; warps take 256 slots at a time.
  auto add_scores = [&](int x, int64_t unit, int count) {
    constexpr int U = 2;  // times 4 slots a thread, their loads together
    float* mass = a.mass + unit * a.M;
    const float4* sc = reinterpret_cast<const float4*>(a.scores + unit * a.heads * a.Ms);
    const int quads = (count + 3) >> 2, stride = a.Ms >> 2;
    const bool aligned = (a.M & 3) == 0;  // rows of masses on 16 bytes
    for (;;) {
      int n0 = 0;
      if (lane == 0) n0 = atomicAdd(&job_next[x], 32 * U);
      n0 = __shfl_sync(0xffffffffu, n0, 0);
      if (n0 >= quads) break;
      n0 += lane;
      float v[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int n = (n0 + u * 32) * 4;
        if (aligned) {
          const float4 y = n < count ? *reinterpret_cast<const float4*>(mass + n) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[u][0] = y.x;
          v[u][1] = y.y;
          v[u][2] = y.z;
          v[u][3] = y.w;
        } else {
#pragma unroll
          for (int z = 0; z < 4; ++z) v[u][z] = n + z < count ? mass[n + z] : 0.f;
        }
      }
      for (int h0 = 0; h0 < a.heads; h0 += 4) {
        float4 y[U][4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (h0 + e < a.heads && n0 + u * 32 < quads) y[u][e] = __ldcg(sc + static_cast<int64_t>(h0 + e) * stride + n0 + u * 32);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (h0 + e < a.heads) {
            const float f0 = fin[x][0][h0 + e], f1 = fin[x][1][h0 + e];
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int n = (n0 + u * 32) * 4;  // slots past the count keep what they hold
              if (n < count) v[u][0] += ex2_approx(y[u][e].x - f0) * f1;
              if (n + 1 < count) v[u][1] += ex2_approx(y[u][e].y - f0) * f1;
              if (n + 2 < count) v[u][2] += ex2_approx(y[u][e].z - f0) * f1;
              if (n + 3 < count) v[u][3] += ex2_approx(y[u][e].w - f0) * f1;
            }
          }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int n = (n0 + u * 32) * 4;
        if (aligned) {
          if (n < count) *reinterpret_cast<float4*>(mass + n) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
        } else {
#pragma unroll
          for (int z = 0; z < 4; ++z)
            if (n + z < count) mass[n + z] = v[u][z];
        }
      }
    }
  };

  // part of CTA c0 + c of a shared unit: its second slot where the unit begins, else its first
  auto part_slot = [&](int c0, int c) { return static_cast<int64_t>(c0 + c) * 2 + (c == 0 ? 1 : 0); };
  // o of a shared unit: four channels a thread, the parts in their order
  auto merge_o = [&](int x, int at, int threads) {
    T* out = static_cast<T*>(a.out) + job_out[x];
    const int c0 = job_c0[x], parts = job_parts[x];
    for (int y = at; y < a.heads * (D / 4); y += threads) {
      const int head = y / (D / 4);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int c = 0; c < parts; ++c) {
        const float4 po = __ldcg(reinterpret_cast<const float4*>(a.part_o + part_slot(c0, c) * HN * D) + y);
        const float f = weights_sh[c * HN + head];
        o.x += f * po.x;
        o.y += f * po.y;
        o.z += f * po.z;
        o.w += f * po.w;
      }
      const float inv = fin[x][1][head];
      T* dst = out + head * a.oh + (y % (D / 4)) * 4;
      dst[0] = T(o.x * inv);
      dst[1] = T(o.y * inv);
      dst[2] = T(o.z * inv);
      dst[3] = T(o.w * inv);
    }
  };

  if (warp > AT_WARPS) {
    const int at = tid - 32 * (AT_WARPS + 1);
    bool told = false;  // the tile warps, whether the last unit is done
    for (int job = 0;; ++job) {
      const int x = job & 1;
      // of one mind: a warp that gave up takes the others along
      if (!finish_barrier_and(warp_wait(&job_full[x], static_cast<uint32_t>((job >> 1) & 1)))) {
        if (lane == 0) report(a.status, LINATTN_DEV_TIMEOUT);
        break;
      }
      const int64_t unit = job_unit[x];
      const int count = job_count[x], c0 = job_c0[x], parts = job_parts[x];
      const bool last = job_last[x] != 0;
      auto slot = [&](int c) { return part_slot(c0, c); };
      bool finish = true;
      if (parts > 1) {
        if (at == 0) {
          __threadfence();  // the tile warps' part before the arrival
          const int n = atomicAdd(a.ticket + unit, 1);
          if (n == parts - 1) a.ticket[unit] = 0;
          __threadfence();
          arrived = n;
        }
        finish_barrier();
        finish = arrived == parts - 1;
        if (finish)
          for (int head = warp - (AT_WARPS + 1); head < a.heads; head += AT_FINISH / 32) {  // lanes over the parts
            float mc[AT_PARTS / 32], lc[AT_PARTS / 32], mx = -INFINITY, sum = 0.f;
#pragma unroll
            for (int y = 0; y < AT_PARTS / 32; ++y) {
              const int c = lane + 32 * y;
              mc[y] = c < parts ? __ldcg(a.part_ml + slot(c) * 2 * HN + head) : -INFINITY;
              lc[y] = c < parts ? __ldcg(a.part_ml + slot(c) * 2 * HN + HN + head) : 0.f;
              mx = fmaxf(mx, mc[y]);
            }
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
#pragma unroll
            for (int y = 0; y < AT_PARTS / 32; ++y) {
              const float f = mc[y] == -INFINITY ? 1.f : ex2_approx(mc[y] - mx);  // scores of NaN only: m = -inf, l = NaN
              sum += f * lc[y];
              if (lane + 32 * y < parts) weights_sh[(lane + 32 * y) * HN + head] = f;
            }
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) {
              fin[x][0][head] = mx == -INFINITY ? 0.f : mx;
              fin[x][1][head] = sum != 0.f ? 1.f / sum : 0.f;
            }
          }
        finish_barrier();
      }
      if (last) {
        if (at == 0) help = finish ? 1 : 0;
        asm volatile("barrier.cta.sync 2, 384;" ::: "memory");
        told = true;
      }
      if (finish && parts > 1) merge_o(x, at, last ? AT_THREADS - 32 : AT_FINISH);
      if (finish && a.accumulate) {
        if (job_tmem[x]) {
          tc_fence_after();
          add_tmem(x, unit, count, 0, last ? 3 : 1);
          tc_fence_before();
        } else {
          add_scores(x, unit, count);
        }
      }
      mbar_arrive(&job_empty[x]);
      if (last) break;
    }
    if (!told) {
      if (at == 0) help = 0;
      asm volatile("barrier.cta.sync 2, 384;" ::: "memory");
    }
    tc_fence_before();
    asm volatile("barrier.cta.sync 2, 384;" ::: "memory");  // the other warps have read their scores
    if (warp == AT_WARPS + 1 && a.accumulate) free_tmem();
    return;
  }

  const int g = lane >> 2, tig = lane & 3;
  const int ct = warp % CT, th = warp / CT;      // P V: 16-channel tile, slots (D = 64: half) of a tile
  constexpr int KT = D == 64 ? 4 : 8;            // 16-slot steps of P V
  const uint32_t ring_a = smem_u32(ring), p_a = smem_u32(pbuf);
  // ldmatrix rows of this lane: K rows 16 warp + ..., V rows by step, P rows by head
  const int krow = 16 * warp + (lane & 15), kchunk = lane >> 4;
  const int vrow = (lane & 7) + ((lane >> 4) & 1) * 8, vchunk = ct * 2 + ((lane >> 3) & 1);
  const uint32_t k_off = krow * 128, v_off = HALVES * SM::HALF + (vchunk >> 3) * SM::HALF;
  int j = 0, jobs = 0;
  bool ok = true;
  // room for a unit's result: the finishing warps are done with the one before the last
  auto job_room = [&] {
    if (jobs >= 2 && ok)
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&job_empty[jobs & 1], static_cast<uint32_t>((jobs / 2 - 1) & 1)));
    tc_fence_after();
  };
  // q as the B operand: channels 16 kk + 2 tig (+ 1, + 8, + 9) of head g
  uint32_t q[NT][D / 16][2];
  auto load_q = [&] {
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const int head = x * 8 + g;
      const T* src = static_cast<const T*>(a.q) + w.b * a.qb + (static_cast<int64_t>(w.h) * a.G + a.h0 + head) * a.qh + 2 * tig;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int e = 0; e < 2; ++e) q[x][kk][e] = head < a.heads ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + e * 8) : 0u;
    }
  };
  load_q();
  for (int64_t t = t0; t < t1;) {
    const int end = static_cast<int>(lmin(w.tiles, first + (t1 - t))), count = w.count;
    const bool whole = first == 0 && end == w.tiles;  // else several CTAs share the unit
    const bool begins = first == 0;
    const bool last = t + (end - first) >= t1;        // of this CTA
    const int64_t unit = static_cast<int64_t>(w.b) * a.H + w.h;
    const int64_t out_at = w.b * a.ob + (static_cast<int64_t>(w.h) * a.G + a.h0) * a.oh;
    float acc[NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      acc[x][0] = acc[x][1] = acc[x][2] = acc[x][3] = 0.f;
      m[x][0] = m[x][1] = -INFINITY;
      l[x][0] = l[x][1] = 0.f;
    }
    float* sc = a.scores + unit * a.heads * a.Ms;
    const int64_t u0 = t - first, u1 = u0 + w.tiles;                       // the unit's tiles among all
    const int64_t c0 = ((u0 + 1) * nc - 1) / total, c1 = (u1 * nc - 1) / total;  // the CTAs that share it
    const bool in_tmem = a.accumulate && whole && w.tiles * NT <= 32 && NT <= 2;
    if (in_tmem) job_room();
    const uint32_t sc_tmem = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + (jobs & 1) * 256 + (warp >> 2) * 128;
    for (int i = first; i < end; ++i, ++j) {
      const int st = j % ST, valid = min(AT_ROWS, count - i * AT_ROWS);
      // a warp whose wait gave up goes on through the barriers
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[st], static_cast<uint32_t>((j / ST) & 1)));
      const uint32_t stage = ring_a + st * SM::STAGE;
      float s[NT][4], s2[NT][4];  // two chains of products
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[x][e] = s2[x][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t f[4];
        const int chunk = (kk & 3) * 2 + kchunk;
        ldsm_x4(stage + (kk >> 2) * SM::HALF + k_off + ((chunk ^ (krow & 7)) << 4), f[0], f[1], f[2], f[3]);
#pragma unroll
        for (int x = 0; x < NT; ++x) M::mma((kk & 1) ? s2[x] : s[x], f, q[x][kk][0], q[x][kk][1]);
      }
      const int r0 = 16 * warp + g, r1 = r0 + 8;
      bool grow = false;
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = e < 2 ? r0 : r1;
          const float v = r < valid ? (s[x][e] + s2[x][e]) * a.scale_log2 : -INFINITY;
          s[x][e] = v;
          grow |= v > m[x][e & 1] + 8.f;
        }
      if (in_tmem) {
#pragma unroll
        for (int x = 0; x < NT; ++x) tmem_st4(sc_tmem + (i * NT + x) * 4, s[x]);
      } else if (a.accumulate) {
        float* row = sc + 2 * tig * a.Ms + i * AT_ROWS + r0;
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            if (x * 8 + 2 * tig + c < a.heads) {
              if (r0 < valid) row[(x * 8 + c) * a.Ms] = s[x][c];
              if (r1 < valid) row[(x * 8 + c) * a.Ms + 8] = s[x][c + 2];
            }
      }
      uint8_t* pb = pbuf + (j & 1) * (2 * HN * AT_PROW);
      float ps[NT][2];  // this lane's share of the tile's sums
      auto weights = [&] {
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          const float z0 = m[x][0] == -INFINITY ? 0.f : m[x][0], z1 = m[x][1] == -INFINITY ? 0.f : m[x][1];
          const float p0 = ex2_approx(s[x][0] - z0), p1 = ex2_approx(s[x][1] - z1);
          const float p2 = ex2_approx(s[x][2] - z0), p3 = ex2_approx(s[x][3] - z1);
          ps[x][0] = p0 + p2;
          ps[x][1] = p1 + p3;
          const uint32_t h01 = M::pack(p0, p1), h23 = M::pack(p2, p3);
          const float2 u01 = M::unpack(h01), u23 = M::unpack(h23);
          // transposed: head g, slots 2 tig and 2 tig + 1
          uint8_t* row = pb + (x * 8 + g) * AT_PROW + (16 * warp + 2 * tig) * 2;
          *reinterpret_cast<uint32_t*>(row) = movmatrix_t(h01);
          *reinterpret_cast<uint32_t*>(row + 16) = movmatrix_t(h23);
          *reinterpret_cast<uint32_t*>(row + HN * AT_PROW) = movmatrix_t(M::pack(p0 - u01.x, p1 - u01.y));
          *reinterpret_cast<uint32_t*>(row + HN * AT_PROW + 16) = movmatrix_t(M::pack(p2 - u23.x, p3 - u23.y));
        }
      };
      weights();
      if (attend_barrier_or(grow)) {  // the running maximum moves only past a margin of 2^8
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float v = fmaxf(s[x][c], s[x][c + 2]);
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
            if (g == 0) mx_w[warp][x * 8 + 2 * tig + c] = v;
          }
        attend_barrier();
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float v = m[x][c];
#pragma unroll
            for (int y = 0; y < AT_WARPS; ++y) v = fmaxf(v, mx_w[y][x * 8 + 2 * tig + c]);
            const float f = m[x][c] == -INFINITY ? 0.f : ex2_approx(m[x][c] - v);
            m[x][c] = v;
            l[x][c] *= f;
            acc[x][c] *= f;
            acc[x][c + 2] *= f;
          }
        weights();
        attend_barrier();
      }
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        l[x][0] += ps[x][0];
        l[x][1] += ps[x][1];
      }
      // O^T += V^T P^T, the lo parts in a chain of their own
      float low[NT][4];
#pragma unroll
      for (int x = 0; x < NT; ++x) low[x][0] = low[x][1] = low[x][2] = low[x][3] = 0.f;
      const uint32_t prow = p_a + (j & 1) * (2 * HN * AT_PROW) + (lane & 7) * AT_PROW + th * KT * 32 + (lane >> 3) * 16;
#pragma unroll
      for (int k2 = 0; k2 < KT / 2; ++k2) {  // 32 slots
        uint32_t f[2][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = (th * KT + 2 * k2 + e) * 16 + vrow;
          ldsm_x4_t(stage + v_off + r * 128 + (((vchunk & 7) ^ (r & 7)) << 4), f[e][0], f[e][1], f[e][2], f[e][3]);
          if (valid < AT_ROWS) {  // slots that are not in use may hold anything: 0 x Inf
            const int s0 = (th * KT + 2 * k2 + e) * 16 + 2 * tig;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int sl = s0 + (y >> 1) * 8;
              f[e][y] &= sl + 1 < valid ? 0xffffffffu : sl < valid ? 0xffffu : 0u;
            }
          }
        }
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          uint32_t b[4];
          ldsm_x4(prow + x * 8 * AT_PROW + k2 * 64, b[0], b[1], b[2], b[3]);
          M::mma(acc[x], f[0], b[0], b[1]);
          M::mma(acc[x], f[1], b[2], b[3]);
          ldsm_x4(prow + (HN + x * 8) * AT_PROW + k2 * 64, b[0], b[1], b[2], b[3]);
          M::mma(low[x], f[0], b[0], b[1]);
          M::mma(low[x], f[1], b[2], b[3]);
        }
      }
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[x][e] += low[x][e];
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
    // ---- the unit's part is done: the next one's q on its way, sums over the warps
    t += end - first;
    first = 0;
    w.next();
    if (!last) load_q();
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) l[x][c] += __shfl_xor_sync(0xffffffffu, l[x][c], o);
        if (g == 0) l_w[warp][x * 8 + 2 * tig + c] = l[x][c];
      }
    if (D == 64 && th == 1) {
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) upper[((ct * 32 + lane) * NT + x) * 4 + e] = acc[x][e];
    }
    attend_barrier();
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float v = 0.f;
#pragma unroll
        for (int y = 0; y < AT_WARPS; ++y) v += l_w[y][x * 8 + 2 * tig + c];
        l[x][c] = v;
      }
    if (D == 64 && th == 0) {
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[x][e] += upper[((ct * 32 + lane) * NT + x) * 4 + e];
    }
    if (in_tmem) {
      tmem_wait_st();
      tc_fence_before();
    } else {
      job_room();
    }
    if (whole) {
      if (warp == 0 && g == 0) {
        float (*result)[HN] = fin[jobs & 1];
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            result[0][x * 8 + 2 * tig + c] = m[x][c] == -INFINITY ? 0.f : m[x][c];
            result[1][x * 8 + 2 * tig + c] = l[x][c] != 0.f ? 1.f / l[x][c] : 0.f;
          }
      }
      if (th == 0) {
        T* out = static_cast<T*>(a.out) + out_at;
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int head = x * 8 + 2 * tig + (e & 1);
            const float inv = l[x][e & 1] != 0.f ? 1.f / l[x][e & 1] : 0.f;
            if (head < a.heads) out[head * a.oh + ct * 16 + g + (e >> 1) * 8] = T(acc[x][e] * inv);
          }
      }
    } else {
      // slot 0: the unit began in an earlier CTA's share
      const int64_t at = static_cast<int64_t>(blockIdx.x) * 2 + (begins ? 1 : 0);
      float* po = a.part_o + at * HN * D;
      float* pml = a.part_ml + at * 2 * HN;
      if (th == 0) {
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) po[(x * 8 + 2 * tig + (e & 1)) * D + ct * 16 + g + (e >> 1) * 8] = acc[x][e];
      }
      if (warp == 0 && g == 0) {
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            pml[x * 8 + 2 * tig + c] = m[x][c];
            pml[HN + x * 8 + 2 * tig + c] = l[x][c];
          }
      }
    }
    attend_barrier();
    if (tid == 0) {
      const int x = jobs & 1;
      job_unit[x] = unit;
      job_out[x] = out_at;
      job_count[x] = count;
      job_c0[x] = static_cast<int>(c0);
      job_parts[x] = whole ? 1 : static_cast<int>(c1 - c0) + 1;
      job_tmem[x] = in_tmem ? 1 : 0;
      job_next[x] = 0;
      job_last[x] = last ? 1 : 0;
      mbar_arrive(&job_full[x]);
    }
    if (last && a.accumulate && t1 - t0 > 8) {
      // meanwhile what the masses need comes to L2, from where longer shares of tiles have pushed it
      // (12 sequences x 8 heads x 4096 slots 47.0 us, without 49.5; shorter ones lose 0.4)
      const int lines = (count + 31) >> 5, rows = in_tmem ? 1 : 1 + a.heads;
      for (int y = tid; y < rows * lines; y += 32 * AT_WARPS) {
        const int head = y / lines, n = (y - head * lines) * 32;
        const float* at = head == 0 ? a.mass + unit * a.M + n : sc + static_cast<int64_t>(head - 1) * a.Ms + n;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
      }
    }
    ++jobs;
  }
  asm volatile("barrier.cta.sync 2, 384;" ::: "memory");
  if (help) {  // with the last unit
    const int x = (jobs - 1) & 1;
    if (job_parts[x] > 1) merge_o(x, AT_FINISH + tid, AT_THREADS - 32);
    if (a.accumulate) {
      tc_fence_after();
      if (job_tmem[x]) add_tmem(x, job_unit[x], job_count[x], 1 + (warp >> 2), 3);
      else add_scores(x, job_unit[x], job_count[x]);
      tc_fence_before();
    }
  }
  asm volatile("barrier.cta.sync 2, 384;" ::: "memory");
  if (!ok && lane == 0) {
    report(a.status, LINATTN_DEV_TIMEOUT);
    dead = 1;
  }
}

int attend_fail(int code, const char* what) {
  char msg[256];
  snprintf(msg, sizeof(msg), "heavy_attend: %s", what);
  return set_error(code, msg);
}

constexpr int AT_HEADS = 32;  // query heads of a group in one launch

int attend_nt(int64_t heads) { return heads > 16 ? 4 : heads > 8 ? 2 : 1; }

template <typename T, int D, int NT>
cudaError_t launch_attend(const HeavyAttendArgs& a, const CUtensorMap& k, const CUtensorMap& v, unsigned grid, cudaStream_t st) {
  auto kern = heavy_attend_kernel<T, D, NT>;
  static int allowed[64] = {};
  const cudaError_t e = allow_smem(kern, AttendSmem<D, NT>::BYTES, allowed);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(AT_THREADS);
  cfg.dynamicSmemBytes = AttendSmem<D, NT>::BYTES;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a, k, v);
}

template <typename T, int D>
cudaError_t dispatch_attend(const HeavyAttendArgs& a, const CUtensorMap& k, const CUtensorMap& v, unsigned grid, cudaStream_t st) {
  const int nt = attend_nt(a.heads);
  return nt == 1 ? launch_attend<T, D, 1>(a, k, v, grid, st)
                 : nt == 2 ? launch_attend<T, D, 2>(a, k, v, grid, st) : launch_attend<T, D, 4>(a, k, v, grid, st);
}

}  // namespace

}  // namespace linattn

using namespace linattn;

namespace {

int64_t attend_ctas(int64_t units, int64_t budget) { return lmin(lmin(sm_count(), AT_PARTS), units * ((budget + AT_ROWS - 1) / AT_ROWS)); }

}  // namespace

extern "C" int64_t linattn_heavy_attend_workspace(int64_t batch, int64_t Hq, int64_t Hkv, int64_t budget) {
  if (batch < 1 || Hkv < 1 || Hq < Hkv || budget < 1) return 0;
  const int64_t heads = lmin(Hq / Hkv, AT_HEADS), hn = 8 * attend_nt(heads);
  return batch * Hkv * heads * ((budget + 3) / 4 * 4) * 4 + sm_count() * 2 * hn * (128 + 2) * 4 + 64;
}

namespace {

bool attend_maps(const linattn_heavy_t* cache, CUtensorMap* tk, CUtensorMap* tv) {
  const int64_t D = cache->head_dim, rows = static_cast<int64_t>(cache->batch) * cache->n_kv_heads * cache->budget;
  const CUtensorMapDataType cu = cache->dtype == LINATTN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const int64_t dims[3] = {D, rows, 1}, strides[2] = {D * 2, rows * D * 2};
  const int box[3] = {64, AT_BOX, 1};
  return tensor_map_3d(tk, cache->k, cu, dims, strides, box) && tensor_map_3d(tv, cache->v, cu, dims, strides, box);
}

// what both entry points ask of a cache
int attend_cache(const linattn_heavy_t* cache) {
  if (!cache || !cache->k || !cache->v || !cache->mass || !cache->seen) return attend_fail(LINATTN_EINVAL, "NULL pointer");
  if (cache->dtype != LINATTN_F16 && cache->dtype != LINATTN_BF16)
    return attend_fail(LINATTN_EUNSUPPORTED, "f16 or bf16 caches");
  if (cache->head_dim != 64 && cache->head_dim != 128) return attend_fail(LINATTN_EUNSUPPORTED, "head_dim must be 64 or 128");
  if (cache->batch < 1 || cache->n_kv_heads < 1 || cache->budget < 1 || cache->budget > (1 << 24))
    return attend_fail(LINATTN_EINVAL, "batch, n_kv_heads and budget must be > 0 (budget <= 2^24)");
  if ((reinterpret_cast<uintptr_t>(cache->k) | reinterpret_cast<uintptr_t>(cache->v) | reinterpret_cast<uintptr_t>(cache->mass)) % 16)
    return attend_fail(LINATTN_EINVAL, "K, V and mass must be 16-byte aligned");
  if (static_cast<int64_t>(cache->batch) * cache->n_kv_heads * cache->budget >= (int64_t(1) << 31))
    return attend_fail(LINATTN_EUNSUPPORTED, "too many slots for 32-bit TMA coordinates");
  return LINATTN_OK;
}

}  // namespace

extern "C" int linattn_heavy_maps(const linattn_heavy_t* cache, void* maps) {
  if (const int rc = attend_cache(cache)) return rc;
  if (!maps) return attend_fail(LINATTN_EINVAL, "NULL pointer");
  static_assert(2 * sizeof(CUtensorMap) == LINATTN_HEAVY_MAPS, "two tensor maps");
  CUtensorMap m[2];
  if (!attend_maps(cache, &m[0], &m[1])) return attend_fail(LINATTN_ECUDA, "tensor map encoding failed");
  memcpy(maps, m, sizeof(m));
  return LINATTN_OK;
}

extern "C" int linattn_heavy_attend(const linattn_heavy_t* cache, const void* q, int64_t Hq, const int64_t* q_strides,
                                    float scale, int32_t accumulate, void* out, const int64_t* out_strides,
                                    int32_t* ticket, void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  if (const int rc = attend_cache(cache)) return rc;
  if (!q || !out || !q_strides || !out_strides || !ticket) return attend_fail(LINATTN_EINVAL, "NULL pointer");
  const int64_t D = cache->head_dim;
  if (Hq < 1 || Hq % cache->n_kv_heads) return attend_fail(LINATTN_EINVAL, "H_q must be a multiple of H_kv");
  if (!(scale > 0.f) || scale > 1e30f) return attend_fail(LINATTN_EINVAL, "scale must be positive and finite");
  if (reinterpret_cast<uintptr_t>(q) % 4 || q_strides[0] % 2 || q_strides[1] % 2)
    return attend_fail(LINATTN_EINVAL, "q rows must be 4-byte aligned");
  const int64_t units = static_cast<int64_t>(cache->batch) * cache->n_kv_heads;
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 ||
      workspace_bytes < linattn_heavy_attend_workspace(cache->batch, Hq, cache->n_kv_heads, cache->budget))
    return attend_fail(LINATTN_EINVAL, "workspace too small or not 16-byte aligned");
  CUtensorMap m[2];
  if (cache->maps) memcpy(m, cache->maps, sizeof(m));
  else if (!attend_maps(cache, &m[0], &m[1])) return attend_fail(LINATTN_ECUDA, "tensor map encoding failed");
  const CUtensorMap &tk = m[0], &tv = m[1];
  HeavyAttendArgs a;
  a.mass = cache->mass;
  a.seen = cache->seen;
  a.q = q;
  a.out = out;
  a.qb = q_strides[0];
  a.qh = q_strides[1];
  a.ob = out_strides[0];
  a.oh = out_strides[1];
  a.B = cache->batch;
  a.H = cache->n_kv_heads;
  a.M = cache->budget;
  a.Ms = (cache->budget + 3) / 4 * 4;
  a.G = static_cast<int>(Hq / cache->n_kv_heads);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.accumulate = accumulate ? 1 : 0;
  a.ticket = ticket;
  a.status = status;
  const unsigned grid = static_cast<unsigned>(attend_ctas(units, cache->budget));
  const int64_t most = lmin(a.G, AT_HEADS), hn = 8 * attend_nt(most);
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + sm_count() * 2 * hn * D;
  a.scores = a.part_ml + sm_count() * 2 * 2 * hn;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  for (a.h0 = 0; e == cudaSuccess && a.h0 < a.G; a.h0 += AT_HEADS) {  // larger groups: 32 heads at a time
    a.heads = static_cast<int>(lmin(a.G - a.h0, AT_HEADS));
    if (cache->dtype == LINATTN_F16) e = D == 128 ? dispatch_attend<__half, 128>(a, tk, tv, grid, st) : dispatch_attend<__half, 64>(a, tk, tv, grid, st);
    else e = D == 128 ? dispatch_attend<__nv_bfloat16, 128>(a, tk, tv, grid, st) : dispatch_attend<__nv_bfloat16, 64>(a, tk, tv, grid, st);
  }
  return e == cudaSuccess ? LINATTN_OK : attend_fail(LINATTN_ECUDA, cudaGetErrorString(e));
}
