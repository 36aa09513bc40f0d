// The choice of beam search, on the device: of every group of B beams the K pairs (beam, token) with the largest summed
// log-probability, in descending order, the lowest beam * V + token first among equals.
//
//   key(b, v) = score[b] + ((z[b, v] - max_b) - log sum_v exp(z[b, v] - max_b))
//
// A logit that is -inf or no number is never chosen and adds nothing to the sum; a score that is -inf or no number marks a
// place without a beam; where the largest logit is infinite, the entries that reach it share the probability.  Keys are 64-bit: a
// 32-bit sum of a score near -100 and a logit makes neighbouring logits equal.  Scores come and go as 32-bit numbers, alone or with what
// they leave of the 64-bit sum as a second one (together 48 bits): a search that hands one choice's scores to the next as 32-bit numbers
// alone rounds at the size of the whole sum with every token (1,000 tokens of 3 nats: off by 1e-3, more than many beams are apart).
// The terms of the sum are 32-bit exponentials; four that lie side by side are added in 32-bit (two roundings of 2^-24), the rest in
// 64-bit: a logarithm of a sum, and so the distance of keys of two beams, is good to 2^-21.
//
// Two kernels.  beam_stats_kernel crosses the logits once: a wavefront takes 512 or 1,024 logits of a row and leaves their maximum
// and sum, and the largest of each segment of 64 or 256.  beam_choose_kernel, one workgroup a group, works on what is left, by a bound
// that K entries surely reach: the best segments of n groups of segments are n entries, and the K-th best of them is such a bound (about K + K^2 / 2n
// segments reach it).  It reads the segments that reach it again; the entries that do are cut down by bounds of the same
// kind until they are few, and put in order by counting, for each, those in front of it.  A bound is a key and a place, so that equal logits
// are cut down too; where more entries reach the first one than the list holds, it is searched bit by bit.
// us, first and second kernel: 32 x 8 beams, vocabulary 131,071 26.2 (5.1 TB/s) and 9.6; 8 x 8, 50,257 5.5 and 8.0; 1 x 4 2.6 and 6.3.  The second is a chain
// of eight barriers and three round trips to memory in one workgroup a group, whatever the logits (one beam far ahead, all equal, in order: within 8 us of it).
// Above 32 candidates the groups of threads are smaller, and each thread counts more of them: both kernels, 50,257, 1 x 16 beams and 32 candidates 14.0,
// 1 x 32 and 64 21.9, 4 x 32 and 64 27.0, 1 x 64 and 128 42.1.
#include "common.h"

#define BEAM_MAX 64              // beams of a group
#define BEAM_MAX_KEEP 128        // candidates of a group
#define LOAD 256                 // logits of a wavefront's load: 64 lanes, 4 each
#define LOADS_FEW 2              // of a wavefront: few logits, or many
#define LOADS_MANY 4
#define STATS_WAVES 4
#define CHOOSE_THREADS 1024
#define CHOOSE_WAVES (CHOOSE_THREADS / DA_WAVE)
#define SHORT_SEGS 2048          // segments of a group up to which they are short
#define SIDES_HELD 2             // loads of segments' entries whose keys a wavefront keeps
#define SEG_LIST 512             // segments that are read again
#define LIST 4096                // their entries that reach the bound
#define LIST_A_THREAD (LIST / CHOOSE_THREADS)

// a 64-bit number that orders like the key; 0 for one that is never chosen
__device__ __forceinline__ uint64_t ordered64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return !(v > -INFINITY) ? 0 : ((u >> 63) ? ~u : (u | 0x8000000000000000ull));
}
__device__ __forceinline__ double unordered64(uint64_t k) {
  return __builtin_bit_cast(double, (k >> 63) ? (k & 0x7fffffffffffffffull) : ~k);
}

__device__ __forceinline__ float clean(float z) { return z == z ? z : -INFINITY; }

typedef float float4_any __attribute__((ext_vector_type(4), aligned(4)));

// e^x of -200 <= x <= 0, a unit in the last place off: the product with log2 e in two parts
__device__ __forceinline__ float exp_near(float x) {
  const float hi = 1.44269502f, lo = 1.92596299e-8f;
  const float p = x * hi, rest = fmaf(x, lo, fmaf(x, hi, -p)), r = __builtin_amdgcn_exp2f(p);
  return fmaf(r, rest * 0.693147181f, r);
}

template <int LOADS, int SEG>    // of a wavefront; logits of a segment
__global__ void __launch_bounds__(STATS_WAVES * DA_WAVE)
beam_stats_kernel(const float* __restrict__ logits, long ldl, int V, int n_segs, int n_parts, float* __restrict__ seg_max,
                  float* __restrict__ part_max, double* __restrict__ part_sum) {
  const int lane = threadIdx.x % DA_WAVE, part = blockIdx.x * STATS_WAVES + threadIdx.x / DA_WAVE, row = blockIdx.y;
  if (part >= n_parts) return;
  const float* z = logits + (size_t)row * ldl;
  const int v0 = part * LOADS * LOAD;
  float x[LOADS][4];
  if (v0 + LOADS * LOAD <= V) {
#pragma unroll
    for (int s = 0; s < LOADS; ++s) {
      const float4_any f = __builtin_nontemporal_load((const float4_any*)(z + v0 + s * LOAD + 4 * lane));
#pragma unroll
      for (int e = 0; e < 4; ++e) x[s][e] = f[e];
    }
  } else {
#pragma unroll
    for (int s = 0; s < LOADS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = v0 + s * LOAD + 4 * lane + e;
        x[s][e] = v < V ? z[v] : -INFINITY;
      }
  }
  float top = -INFINITY, m[LOADS];
#pragma unroll
  for (int s = 0; s < LOADS; ++s) {                       // (the maximum with a number drops what is none)
    m[s] = fmaxf(fmaxf(fmaxf(x[s][0], x[s][1]), fmaxf(x[s][2], x[s][3])), -INFINITY);
    if (SEG == 64) {                                      // 16 lanes
      m[s] = fmaxf(m[s], dpp_move<0xB1, 0xF>(m[s], m[s]));
      m[s] = fmaxf(m[s], dpp_move<0x4E, 0xF>(m[s], m[s]));
      m[s] = fmaxf(m[s], dpp_move<0x141, 0xF>(m[s], m[s]));
      m[s] = fmaxf(m[s], dpp_move<0x140, 0xF>(m[s], m[s]));
    } else {
      m[s] = wave_max(m[s]);
    }
    top = fmaxf(top, m[s]);
  }
  float* row_segs = seg_max + (size_t)row * n_segs;
  if (SEG == 64) {
    top = wave_max(top);
#pragma unroll
    for (int s = 0; s < LOADS; ++s)
      if (lane % 16 == 0 && v0 + s * LOAD + 4 * lane < V) row_segs[(part * LOADS + s) * 4 + lane / 16] = m[s];
  } else {
    float best = m[0];
#pragma unroll
    for (int s = 1; s < LOADS; ++s) best = lane == s ? m[s] : best;
    if (lane < LOADS && v0 + lane * LOAD < V) row_segs[part * LOADS + lane] = best;
  }
  double sum = 0.0;
  const bool infinite = top == INFINITY;
#pragma unroll
  for (int s = 0; s < LOADS; ++s) {
    float e4[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // (what is no number, or -inf, or belongs to a part without entries: -200, whose exponential is 0)
      float d = infinite ? (x[s][e] == top ? 0.f : -200.f) : x[s][e] - top;
      e4[e] = exp_near(fmaxf(d, -200.f));
    }
    sum += (double)((e4[0] + e4[1]) + (e4[2] + e4[3]));
  }
  sum = wave_sum_d(sum);
  if (lane == 0) {
    part_max[(size_t)row * n_parts + part] = top;
    part_sum[(size_t)row * n_parts + part] = sum;
  }
}

struct Chosen {
  uint64_t key;                  // 0: none
  int place;                     // of a segment: its number; of an entry: beam * V + token
};

__device__ __forceinline__ bool in_front(uint64_t key, int place, uint64_t other, int other_place) { return key > other || (key == other && place < other_place); }
__device__ __forceinline__ bool reaches(uint64_t key, int place, const Chosen& bound) { return key > bound.key || (key == bound.key && place <= bound.place); }

template <int CTRL>
__device__ __forceinline__ void best_of_lanes(Chosen& c) {
  const uint32_t lo = (uint32_t)dpp_move_i<CTRL, 0xF>((int)c.key, (int)c.key), hi = (uint32_t)dpp_move_i<CTRL, 0xF>((int)(c.key >> 32), (int)(c.key >> 32));
  const uint64_t k = (uint64_t)hi << 32 | lo;
  const int p = dpp_move_i<CTRL, 0xF>(c.place, c.place);
  if (in_front(k, p, c.key, c.place)) { c.key = k; c.place = p; }
}
// over groups of 4, 8 or 16 lanes
__device__ __forceinline__ int sum_of_lanes(int v, int lanes) {
  v += dpp_move_i<0xB1, 0xF>(v, v);
  v += dpp_move_i<0x4E, 0xF>(v, v);
  if (lanes >= 8) v += dpp_move_i<0x141, 0xF>(v, v);
  if (lanes >= 16) v += dpp_move_i<0x140, 0xF>(v, v);
  return v;
}

// Every thread's best entry: the K-th best of the best entries of groups of `lanes` threads goes to bounds[0] (which keeps what it
// holds where fewer groups have any), the best to bounds[1].
__device__ __forceinline__ void bound_of(Chosen best, int lanes, int K, Chosen* group_best, Chosen* bounds) {
  const int t = threadIdx.x, n_groups = CHOOSE_THREADS / lanes;
  best_of_lanes<0xB1>(best);
  best_of_lanes<0x4E>(best);
  if (lanes >= 8) best_of_lanes<0x141>(best);
  if (lanes >= 16) best_of_lanes<0x140>(best);
  if (t % lanes == 0) group_best[t / lanes] = best;
  __syncthreads();
  int before = 0;                                       // the threads of a group count, each its part, the groups in front of it
#pragma unroll 4
  for (int j = t % lanes; j < n_groups; j += lanes) {
    const Chosen other = group_best[j];
    before += in_front(other.key, other.place, best.key, best.place) || (other.key == best.key && other.place == best.place && j < t / lanes);
  }
  before = sum_of_lanes(before, lanes);
  if (before == K - 1 && best.key) bounds[0] = best;    // (the threads of a group write the same)
  if (before == 0) bounds[1] = best;
  __syncthreads();
}

// A bound that `keep` entries reach moved up until at most `most` do: first its key, between it and the largest one, then, where
// more are equal, its place.  count(bound): how many reach it, the same in all threads.
template <class Count>
__device__ void narrow(Chosen& bound, uint64_t largest, int keep, int most, Count count) {
  uint64_t hi = largest + 1;                            // fewer than `keep` reach it
  int c = most + 1;
  while (c > most && hi - bound.key > 1) {
    const uint64_t mid = bound.key + (hi - bound.key) / 2;
    const int m = count(Chosen{mid, 0x7fffffff});
    if (m >= keep) { bound = Chosen{mid, 0x7fffffff}; c = m; }
    else hi = mid;
  }
  if (c <= most) return;
  for (int a = 0; a < bound.place;) {
    const int mid = a + (bound.place - a) / 2;
    if (count(Chosen{bound.key, mid}) >= keep) bound.place = mid;
    else a = mid + 1;
  }
}

// magic: 2^32 / n_segs rounded up (0: divide), for fewer than 65,536 segments
// HELD: segments whose keys a thread keeps (those behind them it works out again)
template <int SEG, int HELD>
__global__ void __launch_bounds__(CHOOSE_THREADS)
beam_choose_kernel(const float* __restrict__ logits, long ldl, int V, int B, int K, const float* __restrict__ scores,
                   const float* __restrict__ scores_low, int n_segs, int n_parts, const float* __restrict__ seg_max, const float* __restrict__ part_max, const double* __restrict__ part_sum,
                   float* __restrict__ out_score, float* __restrict__ out_low, int* __restrict__ out_parent, int* __restrict__ out_token,
                   uint32_t magic) {
  constexpr int SEG_LANES = SEG / 4, SIDE = DA_WAVE / SEG_LANES;      // a segment's lanes, 4 entries each; segments of a wavefront side by side
  __shared__ double base[BEAM_MAX], logsum[BEAM_MAX];     // the score (-inf: no beam); the logarithm of the sum
  __shared__ float top[BEAM_MAX];
  __shared__ Chosen group_best[CHOOSE_THREADS / 4], list[LIST], bounds[2];
  __shared__ int segs[SEG_LIST], counts[CHOOSE_WAVES], n_list[2];
  const int g = blockIdx.x, t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t / DA_WAVE), lane = t % DA_WAVE;
  const size_t row0 = (size_t)g * B;
  const int n = B * n_segs;
  const int lanes = K <= 32 ? 16 : (K <= 64 ? 8 : 4);     // of a group: 64, 128 or 256 groups, twice as many as candidates
  // The t-th of what is shared out over the threads: neighbours go to different groups, so that a beam that is ahead of the
  // others has its segments in all of them.
  const int t_of = t % lanes * (CHOOSE_THREADS / lanes) + t / lanes;

  // ---- asked for together: a thread's first segments, and the partial results of the wavefront's first row
  const float* sm = seg_max + row0 * n_segs;
  float zr[HELD];
#pragma unroll
  for (int e = 0; e < HELD; ++e) zr[e] = sm[min(t_of + e * CHOOSE_THREADS, n - 1)];
  for (int b = wave; b < B; b += CHOOSE_WAVES) {
    const float* pm = part_max + (row0 + b) * n_parts;
    const double* ps = part_sum + (row0 + b) * n_parts;
    const double sc = (double)scores[row0 + b] + (scores_low ? (double)scores_low[row0 + b] : 0.0);
    // (a lane past the end takes the last part's maximum again, and no sum)
    const float p0 = pm[min(lane, n_parts - 1)], p1 = pm[min(lane + DA_WAVE, n_parts - 1)];
    const double s0 = ps[min(lane, n_parts - 1)], s1 = ps[min(lane + DA_WAVE, n_parts - 1)];
    float m = fmaxf(p0, p1);
    for (int i = lane + 2 * DA_WAVE; i < n_parts; i += DA_WAVE) m = fmaxf(m, pm[i]);
    m = wave_max(m);
    auto weighed = [&](float p, double s) { return s * (double)expf(p == m ? 0.f : p - m); };      // (a part without entries has the sum 0)
    double s = (lane < n_parts ? weighed(p0, s0) : 0.0) + (lane + DA_WAVE < n_parts ? weighed(p1, s1) : 0.0);
    for (int i = lane + 2 * DA_WAVE; i < n_parts; i += DA_WAVE) s += weighed(pm[i], ps[i]);
    s = wave_sum_d(m > -INFINITY ? s : 0.0);
    if (lane == 0) {
      top[b] = m;
      base[b] = (m > -INFINITY && sc == sc) ? sc : -INFINITY;
      logsum[b] = s > 0.0 ? log(s) : 0.0;
    }
  }
  if (t < 2) n_list[t] = 0;
  if (t < 2) bounds[t] = Chosen{1, 0x7fffffff};           // (every entry that can be chosen reaches it)
  __syncthreads();
  auto key_of = [&](int b, float z) {
    const double x = z == top[b] ? 0.0 : (double)z - (double)top[b];
    return ordered64(base[b] + (x - logsum[b]));
  };
  auto total = [&](int c) {                               // over the workgroup
    c = wave_sum_i(c);
    __syncthreads();
    if (lane == 0) counts[wave] = c;
    __syncthreads();
    c = 0;
    for (int w = 0; w < CHOOSE_WAVES; ++w) c += counts[w];
    return c;
  };
  auto row_of = [&](int i) { return magic ? (int)__umulhi((uint32_t)i, magic) : i / n_segs; };

  // ---- a bound for the segments' largest entries
  uint64_t held[HELD];
  Chosen best{0, 0x7fffffff};
  auto better = [&](uint64_t k, int i) {
    if (in_front(k, i, best.key, best.place)) best = Chosen{k, i};
  };
#pragma unroll
  for (int e = 0; e < HELD; ++e) {
    const int i = t_of + e * CHOOSE_THREADS;
    held[e] = i < n ? key_of(row_of(i), zr[e]) : 0;
    better(held[e], i);
  }
  for (int i = t_of + HELD * CHOOSE_THREADS; i < n; i += CHOOSE_THREADS) better(key_of(row_of(i), sm[i]), i);
  bound_of(best, lanes, K, group_best, bounds);
  Chosen bound = bounds[0];
  const uint64_t largest = bounds[1].key;

  // ---- the segments that reach it
  auto each_seg = [&](auto f) {
#pragma unroll
    for (int e = 0; e < HELD; ++e) f(held[e], t_of + e * CHOOSE_THREADS);      // (one past the end has the key 0)
    for (int i = t_of + HELD * CHOOSE_THREADS; i < n; i += CHOOSE_THREADS) f(key_of(row_of(i), sm[i]), i);
  };
  auto list_segs = [&]() {
    each_seg([&](uint64_t k, int i) {
      if (reaches(k, i, bound)) {
        const int at = atomicAdd(&n_list[0], 1);
        if (at < SEG_LIST) segs[at] = i;
      }
    });
    __syncthreads();
    return n_list[0];
  };
  int n_found = list_segs();
  if (n_found > SEG_LIST) {
    narrow(bound, largest, K, SEG_LIST, [&](const Chosen& at) {
      int c = 0;
      each_seg([&](uint64_t k, int i) { c += reaches(k, i, at); });
      return total(c);
    });
    __syncthreads();
    if (t == 0) n_list[0] = 0;
    __syncthreads();
    n_found = list_segs();
  }
  // As many entries as segments reach the bound that ends with its segment.
  if (bound.place < n) bound.place = min(row_of(bound.place) * V + (bound.place - row_of(bound.place) * n_segs + 1) * SEG - 1, (row_of(bound.place) + 1) * V - 1);

  // ---- their entries that reach it
  auto keys_of = [&](int j, uint64_t k[4]) {              // of 4 entries of the list's segment SIDE j + lane / SEG_LANES; the first one's place
    const int at = SIDE * j + lane / SEG_LANES, i = segs[min(at, n_found - 1)], b = row_of(i), v = (i - b * n_segs) * SEG + 4 * (lane % SEG_LANES);
    const float* z = logits + (row0 + b) * ldl + v;
    float x[4];
    if (at < n_found && v + 4 <= V) {
      const float4_any f = *(const float4_any*)z;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = clean(f[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = at < n_found && v + e < V ? clean(z[e]) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) k[e] = key_of(b, x[e]);
    return b * V + v;
  };
  const int n_sides = (n_found + SIDE - 1) / SIDE;
  uint64_t kept[SIDES_HELD][4];
  int place_kept[SIDES_HELD];
#pragma unroll
  for (int h = 0; h < SIDES_HELD; ++h) {
    place_kept[h] = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) kept[h][e] = 0;
    if (wave + h * CHOOSE_WAVES < n_sides) place_kept[h] = keys_of(wave + h * CHOOSE_WAVES, kept[h]);
  }
  auto each_entry = [&](auto f) {
#pragma unroll
    for (int h = 0; h < SIDES_HELD; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) f(kept[h][e], place_kept[h] + e);
    for (int j = wave + SIDES_HELD * CHOOSE_WAVES; j < n_sides; j += CHOOSE_WAVES) {
      uint64_t k[4];
      const int place = keys_of(j, k);
#pragma unroll
      for (int e = 0; e < 4; ++e) f(k[e], place + e);
    }
  };
  auto list_entries = [&]() {
    each_entry([&](uint64_t k, int place) {
      if (reaches(k, place, bound)) {
        const int at = atomicAdd(&n_list[1], 1);
        if (at < LIST) list[at] = Chosen{k, place};
      }
    });
    __syncthreads();
    return n_list[1];
  };
  int n_entries = list_entries();
  if (n_entries > LIST) {
    narrow(bound, largest, K, LIST, [&](const Chosen& at) {
      int c = 0;
      each_entry([&](uint64_t k, int place) { c += reaches(k, place, at); });
      return total(c);
    });
    __syncthreads();
    if (t == 0) n_list[1] = 0;
    __syncthreads();
    n_entries = list_entries();
  }

  // ---- few of them: by bounds of the same kind (there are more entries than groups, neighbours in different ones: each group has some)
  while (n_entries > CHOOSE_THREADS / lanes * 3 / 2) {
    Chosen mine[LIST_A_THREAD], first{0, 0x7fffffff};
#pragma unroll
    for (int e = 0; e < LIST_A_THREAD; ++e) {
      const int i = t_of + e * CHOOSE_THREADS;
      mine[e] = i < n_entries ? list[i] : Chosen{0, 0x7fffffff};
      if (in_front(mine[e].key, mine[e].place, first.key, first.place)) first = mine[e];
    }
    bound_of(first, lanes, K, group_best, bounds);
    const Chosen next = bounds[0];
    if (t == 0) n_list[1] = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < LIST_A_THREAD; ++e)
      if (mine[e].key && reaches(mine[e].key, mine[e].place, next)) list[atomicAdd(&n_list[1], 1)] = mine[e];
    __syncthreads();
    const int left = n_list[1];
    if (left == n_entries) break;
    n_entries = left;
  }

  // ---- in order: 4 threads an entry count those in front of it
  for (int i0 = 0; i0 < n_entries; i0 += CHOOSE_THREADS / 4) {
    const int i = i0 + t / 4;
    const Chosen mine = list[min(i, n_entries - 1)];
    int r = 0;
#pragma unroll 4
    for (int j = t % 4; j < n_entries; j += 4) r += in_front(list[j].key, list[j].place, mine.key, mine.place);
    r = sum_of_lanes(r, 4);
    if (t % 4 == 0 && i < n_entries && r < K) {
      const double sc = unordered64(mine.key);
      const float near = (float)sc;
      out_score[(size_t)g * K + r] = near;
      if (out_low) out_low[(size_t)g * K + r] = fabsf(near) < INFINITY ? (float)(sc - (double)near) : 0.f;
      out_parent[(size_t)g * K + r] = mine.place / V;
      out_token[(size_t)g * K + r] = mine.place % V;
    }
  }
  if (t >= n_entries && t < K) {
    out_score[(size_t)g * K + t] = -INFINITY;
    if (out_low) out_low[(size_t)g * K + t] = 0.f;
    out_parent[(size_t)g * K + t] = -1;
    out_token[(size_t)g * K + t] = -1;
  }
}

// How a call is cut up.  Short segments while a group's fit the threads that keep their keys: of long ones a small vocabulary has fewer
// than candidates.  Few logits: as many wavefronts as there can be; many: fewer partial results.
struct Cut {
  int seg, loads;
  long n_segs, n_parts;          // of a row
};
static Cut beam_cut(long rows, int B, int V) {
  Cut c;
  c.seg = (long)B * (((long)V + 63) / 64) <= SHORT_SEGS ? 64 : 256;
  c.loads = rows * (((long)V + LOAD - 1) / LOAD) < 16384 ? LOADS_FEW : LOADS_MANY;
  c.n_segs = ((long)V + c.seg - 1) / c.seg;
  c.n_parts = ((long)V + c.loads * LOAD - 1) / (c.loads * LOAD);
  return c;
}

// Scratch of a call, in 32-bit words: the parts' sums (64-bit) and maxima, and the segments' maxima.
extern "C" int da_beam_select_words(int G, int B, int V) {
  if (G < 0 || B <= 0 || V <= 0) return -1;
  const Cut c = beam_cut((long)G * B, B, V);
  const long words = (long)G * B * (3 * c.n_parts + c.n_segs);
  return words > 0x7fffffffL ? -1 : (int)words;
}

// scores_low, out_low: what the scores leave of the 64-bit sums (null: nothing).
extern "C" int da_beam_select_low(const float* logits, long ldl, int G, int B, int V, const float* scores, const float* scores_low, int K,
                                  float* out_score, float* out_low, int* out_parent, int* out_token, float* scratch, long scratch_words,
                                  void* stream) {
  DA_REQUIRE(G >= 0 && B > 0 && B <= BEAM_MAX && V > 0 && ldl >= V && (long)B * V <= 0x7fff0000L,
             "beam_select: bad sizes (groups=%d beams=%d vocabulary=%d row length %ld; at most %d beams)", G, B, V, ldl, BEAM_MAX);
  DA_REQUIRE(K > 0 && K <= BEAM_MAX_KEEP, "beam_select: %d candidates (1 to %d)", K, BEAM_MAX_KEEP);
  if (G == 0) return 0;
  const long rows = (long)G * B;
  const Cut cut = beam_cut(rows, B, V);
  const int n_parts = (int)cut.n_parts, n_segs = (int)cut.n_segs;
  const long words = rows * (3L * n_parts + n_segs);
  DA_REQUIRE(rows <= 65535, "beam_select: %ld rows (at most 65,535)", rows);
  DA_REQUIRE(scratch && (uintptr_t)scratch % 8 == 0 && scratch_words >= words, "beam_select: %ld words of scratch on 8 bytes are needed, found %ld", words, scratch_words);
  double* part_sum = (double*)scratch;
  float* part_max = scratch + 2 * rows * n_parts;
  float* seg_max = part_max + rows * n_parts;
  const dim3 grid(da_ceil_div(n_parts, STATS_WAVES), (unsigned)rows), block(STATS_WAVES * DA_WAVE);
#define DA_STATS(LOADS, SEG) \
  hipLaunchKernelGGL((beam_stats_kernel<LOADS, SEG>), grid, block, 0, (hipStream_t)stream, logits, ldl, V, n_segs, n_parts, seg_max, part_max, part_sum)
  if (cut.seg == 64 && cut.loads == LOADS_FEW) DA_STATS(LOADS_FEW, 64);
  else if (cut.seg == 64) DA_STATS(LOADS_MANY, 64);
  else if (cut.loads == LOADS_FEW) DA_STATS(LOADS_FEW, 256);
  else DA_STATS(LOADS_MANY, 256);
#undef DA_STATS
  DA_CHECK_LAUNCH("beam_select (sums)");
  // i * magic / 2^32 is i / n_segs while i < 2^16 and n_segs < 2^16: the product's error, i * (magic * n_segs - 2^32) / n_segs / 2^32, is below i / 2^32
  const uint32_t magic = (long)B * n_segs < 65536 && n_segs > 1 ? (uint32_t)(((1ull << 32) + n_segs - 1) / n_segs) : 0;
#define DA_CHOOSE(SEG, HELD) \
  hipLaunchKernelGGL((beam_choose_kernel<SEG, HELD>), dim3(G), dim3(CHOOSE_THREADS), 0, (hipStream_t)stream, logits, ldl, V, B, K, scores, scores_low, n_segs, n_parts, \
                     seg_max, part_max, part_sum, out_score, out_low, out_parent, out_token, magic)
  if (cut.seg == 64) DA_CHOOSE(64, 2);
  else if (B * n_segs <= 2 * CHOOSE_THREADS) DA_CHOOSE(256, 2);
  else DA_CHOOSE(256, 4);                               // (32 x 8 beams, 131,071: 34.4 us for 37.1)
#undef DA_CHOOSE
  DA_CHECK_LAUNCH("beam_select (choice)");
  return 0;
}

extern "C" int da_beam_select(const float* logits, long ldl, int G, int B, int V, const float* scores, int K, float* out_score,
                              int* out_parent, int* out_token, float* scratch, long scratch_words, void* stream) {
  return da_beam_select_low(logits, ldl, G, B, V, scores, nullptr, K, out_score, nullptr, out_parent, out_token, scratch, scratch_words, stream);
}
