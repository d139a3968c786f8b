// Tiles of packed sequences: which rows of which sequence a CTA works on, found on the
// device from the offsets, so that no call needs them on the host.
#pragma once

#include "common.cuh"

namespace linattn {

// Rows [first, first + n) of sequence s.  Offsets that are not ascending or leave [0, N]
// are clamped; false if they had to be.
__device__ __forceinline__ bool packed_range(const int32_t* cu, int s, int64_t N, int* first, int* n) {
  const int64_t a = cu[s], b = cu[s + 1];
  const int64_t lo = lmin(lmax(a, 0), N), hi = lmin(lmax(b, lo), N);
  *first = static_cast<int>(lo);
  *n = static_cast<int>(hi - lo);
  return a == lo && b == hi;
}

// Which rows are some sequence's, among its first `most`: the others (padding before the first
// sequence or past the last, holes between clamped offsets, rows beyond the longest sequence that
// the caller named) are never written.  A warp asks for 32 rows in ascending order: `load`
// fetches the offsets of up to 32 sequences, so that it can go out with other loads, and `has`
// answers; of more sequences `has` finds the ones that matter by a search, 32 ways a step.
struct PackedOwner {
  const int32_t* cu;
  int64_t N;
  int S, most, first, n;  // the last two: of this lane's sequence
  __device__ __forceinline__ void fetch(int s) {
    first = n = 0;
    if (s < S) packed_range(cu, s, N, &first, &n);
    n = min(n, most);
  }
  __device__ __forceinline__ void load(const int32_t* offsets, int sequences, int64_t rows, int longest) {
    cu = offsets;
    S = sequences;
    N = rows;
    most = longest;
    fetch(S <= 32 ? threadIdx.x & 31 : S);
  }
  __device__ __forceinline__ bool has(int64_t row) {
    const int lane = threadIdx.x & 31;
    const int64_t lo = __shfl_sync(0xffffffffu, row, 0), hi = __shfl_sync(0xffffffffu, row, 31);
    bool owned = false;
    auto look = [&] {
      unsigned near = __ballot_sync(0xffffffffu, n > 0 && first <= hi && first + n > lo);
      for (; near; near &= near - 1) {
        const int l = __ffs(near) - 1, f = __shfl_sync(0xffffffffu, first, l), c = __shfl_sync(0xffffffffu, n, l);
        owned |= row >= f && row < f + c;
      }
    };
    if (S <= 32) {
      look();
      return owned;
    }
    int s0 = 0;  // the last sequence that begins at or before `lo` is in [s0, s0 + span)
    for (int span = S; span > 32;) {
      const int step = (span + 31) / 32, s = s0 + lane * step;
      const unsigned before = __ballot_sync(0xffffffffu, lane * step < span && cu[min(s, S)] <= lo);
      const int l = before ? 31 - __clz(before) : 0;
      s0 += l * step;
      span = min(step, span - l * step);
    }
    for (; s0 < S; s0 += 32) {
      fetch(s0 + lane);
      look();
      if (__shfl_sync(0xffffffffu, s0 + 32 < S ? first : 0, 31) > hi) break;
    }
    return owned;
  }
};

// The sequence of the `idx`-th tile of `rows` rows of `cu`'s sequences (`most` rows of one at
// most), one after the other: the tile among its sequence's, and the sequence's range in both `cu`
// and `other`.  All lanes of a warp call it and get the same answer.  False past the last tile.
struct PackedTile {
  int tile, first, n, other_first, other_n;
  bool sound;  // no offset had to be clamped
};
__device__ __forceinline__ bool packed_tile(const int32_t* cu, const int32_t* other, int S, int64_t N, int64_t N_other,
                                            int rows, int most, int64_t idx, PackedTile* t) {
  const int lane = threadIdx.x & 31;
  int64_t base = 0;
  for (int s0 = 0; s0 < S; s0 += 32) {
    int first = 0, n = 0, other_first = 0, other_n = 0;
    bool sound = true;
    if (s0 + lane < S) {  // both ranges in one round trip
      sound = packed_range(cu, s0 + lane, N, &first, &n);
      sound &= packed_range(other, s0 + lane, N_other, &other_first, &other_n);
    }
    const int mine = (min(n, most) + rows - 1) / rows;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    if (idx < base + total) {
      const int off = static_cast<int>(idx - base);
      const int l = __ffs(__ballot_sync(0xffffffffu, off >= incl - mine && off < incl)) - 1;
      t->tile = off - __shfl_sync(0xffffffffu, incl - mine, l);
      t->first = __shfl_sync(0xffffffffu, first, l);
      t->n = __shfl_sync(0xffffffffu, n, l);
      t->other_first = __shfl_sync(0xffffffffu, other_first, l);
      t->other_n = __shfl_sync(0xffffffffu, other_n, l);
      t->sound = __shfl_sync(0xffffffffu, sound ? 1 : 0, l) != 0;
      return true;
    }
    base += total;
  }
  return false;
}

// Launch that does not wait for the end of the stream's previous kernel: the kernel starts with
// what needs nothing of others and waits (griddepcontrol.wait) before it reads or writes.
template <typename K, typename... A>
cudaError_t launch_ahead(K kern, dim3 grid, unsigned threads, size_t smem, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace linattn
