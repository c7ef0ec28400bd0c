// Work of many lengths, one after another, cut into equal runs: entry i has steps(i) steps for each
// of `heads` heads, and the steps of all entries, heads within an entry, are numbered through.  A
// CTA counts them itself (the lengths are known to the device alone), and anyone finds the entry,
// head and step of a number.
#pragma once

#include "fk_common.cuh"

namespace fk {

template <int THREADS>
struct RunCount {
  int64_t begins[THREADS + 1];     // steps of one head before the first of a thread's entries
  int64_t warps[THREADS / 32];
};

__host__ __device__ __forceinline__ int entries_of_thread(int n, int threads) {
  return (n + threads - 1) / threads;
}

// By all threads of the CTA; returns the steps of one head before this thread's first entry.
template <int THREADS, class Steps>
__device__ __forceinline__ int64_t count_runs(RunCount<THREADS>& c, int n, Steps steps) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = entries_of_thread(n, THREADS);
  const int a = min((int)threadIdx.x * per, n), b = min(a + per, n);
  int64_t mine = 0;
  for (int i = a; i < b; ++i) mine += steps(i);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) c.warps[warp] = incl;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += c.warps[w];
    total += c.warps[w];
  }
  c.begins[threadIdx.x] = before + incl - mine;
  if (threadIdx.x == 0) c.begins[THREADS] = total;
  __syncthreads();
  return before + incl - mine;
}

// Steps of each of so many equal runs.
__device__ __forceinline__ int64_t run_length(int64_t total, int64_t runs) {
  return total >> 31 ? (total + runs - 1) / runs
                     : (int64_t)(((uint32_t)total + (uint32_t)runs - 1) / (uint32_t)runs);
}

struct RunPlace {
  int entry, head, step;
};

// Place of step x, which is below the number of all; by all lanes of a warp, for the same x.
template <int THREADS, class Steps>
__device__ __forceinline__ RunPlace find_run(const RunCount<THREADS>& c, int n, int heads, int64_t x,
                                             Steps steps) {
  // (32-bit divisions where they do)
  const int64_t at = x >> 31 ? x / heads : (int64_t)((uint32_t)x / (uint32_t)heads);
  // the last thread that begins at or before it, in two rounds of a look by every lane
  constexpr int PER = THREADS / 32;
  const int lane = threadIdx.x & 31;
  const uint32_t group = __ballot_sync(0xffffffffu, c.begins[lane * PER] <= at);
  const int g = (31 - __clz(group)) * PER;
  const uint32_t in_group = __ballot_sync(0xffffffffu, lane < PER && c.begins[g + lane] <= at);
  const int lo = g + 31 - __clz(in_group);
  int64_t before = c.begins[lo];
  RunPlace r;
  r.entry = min(lo * entries_of_thread(n, THREADS), n - 1);
  int s = steps(r.entry);
  while (r.entry + 1 < n && before + s <= at) {
    before += s;
    s = steps(++r.entry);
  }
  s = max(s, 1);
  const int64_t in = x - before * heads;         // below s * heads
  r.head = (int)(in >> 31 ? in / s : (int64_t)((uint32_t)in / (uint32_t)s));
  r.step = (int)(in - (int64_t)r.head * s);
  return r;
}

}  // namespace fk
