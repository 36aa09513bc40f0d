// Attention of one new token a beam over the paged cache, for groups of B sequences that begin with the same pages: the keys
// and values of those pages are read once a group.
//
//   o[r] = sum_j softmax_j(scale q[r] . k[j]) v[j]     over the positions lo_r <= j < len_r of row r's sequence
//
// The rows of a group that meet one key head (its B beams, Hq / Hkv query heads each) are the columns of the matrix products, 16 or
// 32 a workgroup: up to so many rows for the bytes of one.  The positions are walked in chunks of 64: chunks that all rows share, then each
// beam's own ones, of which only that beam's columns take part.  The chunks are shared out over the wavefronts of a workgroup and
// over `splits` workgroups, by the launch's shape and the sequences' lengths; their partial results (weighted sums, maximum, sum of
// weights) are joined in LDS and by a second kernel, in a fixed order.
//
//   scores : S^T[key, row] = K[key, :] . q[row, :], 16 keys a product.  A lane receives 4 keys of one row.
//   softmax: a row's running maximum is the same in the four lanes that hold its keys, its sum is theirs alone until the end.
//   values : O^T[d, row] += V^T[d, key] P^T[key, row].  Values lie dimension by dimension, so the left operand is read as it lies;
//            which key stands in which row of the first product is chosen so that a lane's weights are the ones that the second
//            takes from it: nothing is exchanged.
// bfloat16: a 32-bit weight goes in as three bfloat16 parts, which lose nothing (3 x 8 bits), as in the decode kernel that takes the step
// otherwise: with two, small differences of weights are off by more than the result's rounding, for 1 % (8 x 8 beams over 1,003 positions 17.4 us
// in place of 17.7, 1 x 4 over 531 7.7 in place of 7.8, 4 x 4 over 32,701 the same).  32-bit: 16x16x4 products, nothing is rounded.
// Bound by memory where contexts are long (4 x 4 beams, 32 / 8 heads of 128, 32,701 positions: 101 us, 5.4 TB/s), else by three round trips, lengths,
// pages, keys and values, of which the second travels beside the chunk before.  us: 1 x 4 beams of 12 heads over 531 positions 7.9, 8 x 8 of 25 heads over
// 1,003 17.7; 32-bit, 2 x 5 of 12 heads over 777 10.2 and the joining kernel's 3.1: there a share has too few chunks for 8 wavefronts, and each loads its two
// halves one after the other (the products are a sixth of the time).
#include "gemm_common.h"
#include <da_lane_swap.h>

#define BEAMS_MAX 64             // beams of a group
#define BEAMS_MAX_D 256
#define CHUNK 64
#define TILE 16                  // rows of a matrix product

template <int N>
struct Int { static const int value = N; };
struct Yes { static const bool value = true; };
struct No { static const bool value = false; };

// 2^x: scores carry log2 e in their scale
__device__ __forceinline__ float exp_of_2(float x) { return __builtin_amdgcn_exp2f(x); }

// Over the four lanes that hold a row's keys
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, DA_WAVE));
  return half_max(v);
}

// Over the wavefront, in every lane
template <class Op>
__device__ __forceinline__ int wave_join(int v, Op op) {
  v = op(v, dpp_move_i<0xB1, 0xF>(v, v));
  v = op(v, dpp_move_i<0x4E, 0xF>(v, v));
  v = op(v, dpp_move_i<0x141, 0xF>(v, v));
  v = op(v, dpp_move_i<0x140, 0xF>(v, v));
  v = op(v, dpp_move_i<0x142, 0xA>(v, v));
  v = op(v, dpp_move_i<0x143, 0xC>(v, v));
  return __builtin_amdgcn_readlane(v, DA_WAVE - 1);
}
// the sum of the lanes up to this one
__device__ __forceinline__ int wave_scan(int v) {
  v += dpp_move_i<0x111, 0xF>(0, v);
  v += dpp_move_i<0x112, 0xF>(0, v);
  v += dpp_move_i<0x114, 0xF>(0, v);
  v += dpp_move_i<0x118, 0xF>(0, v);
  v += dpp_move_i<0x142, 0xA>(0, v);
  v += dpp_move_i<0x143, 0xC>(0, v);
  return v;
}

// DK: head size in steps of 32, rounded up to a power of two.  STEP: keys whose loads are under way together.
// RT: tiles of 16 rows.
template <typename T, int DK, int STEP, int WAVES, int RT>
__global__ void __launch_bounds__(WAVES * DA_WAVE)
attn_beams_kernel(const T* __restrict__ q, int q_ld, const T* __restrict__ cache, const int* __restrict__ block_table, int max_blocks,
                  const int* __restrict__ seq_lens, const int* __restrict__ shared, int B, int Hq, int Hkv, int D, int page, float scale,
                  int window, T* __restrict__ out, int out_ld, int splits, float* __restrict__ partial) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int DV = 2 * DK, DMAX = 32 * DK;            // value dimensions in steps of 16
  constexpr int QS = F32 ? 2 * DK : DK;                 // key loads a row: 16 dimensions (32-bit) or 32 (bfloat16) a step
  constexpr int KP = STEP / 16;                         // pieces of 16 keys
  constexpr int VP = F32 ? STEP / 16 : STEP / 32;       // value loads a dimension: 4 keys (32-bit) or 8 a lane
  constexpr int SPAN = F32 ? 4 : 8;                     // consecutive keys of a lane
  constexpr int ROWS = TILE * RT;
  __shared__ float acc_lds[WAVES][DMAX][ROWS + 1];
  __shared__ float m_lds[WAVES][ROWS], l_lds[WAVES][ROWS];

  const int t = threadIdx.x, lane = t % DA_WAVE, wave = __builtin_amdgcn_readfirstlane(t / DA_WAVE);
  const int col = lane % 16, quad = lane / 16;
  const int ratio = Hq / Hkv, R = B * ratio;
  const int hk = blockIdx.x % Hkv, rb = blockIdx.x / Hkv, g = blockIdx.y, z = blockIdx.z;
  const int r0 = rb * ROWS, s0 = g * B;
  const int b0 = r0 / ratio, b1 = (min(r0 + ROWS, R) - 1) / ratio;      // the beams of these rows
  const int lg = 31 - __builtin_clz(page), pmask = page - 1;
  const uint32_t page_elems = 2u * (uint32_t)(Hkv * page * D);
  const int cap = max_blocks * page;                    // (a longer length would lead out of the table)

  // a beam a lane: its length; then the query rows, the right operand (row r of the group is column (r - r0) % 16 of tile (r - r0) / 16)
  const int n_raw = seq_lens[s0 + (lane < B ? lane : 0)], shared_g = shared[g];
  int beam[RT];
  uint4 qf[RT][QS];
#pragma unroll
  for (int y = 0; y < RT; ++y) {
    const int r = r0 + TILE * y + col, rr = min(r, R - 1);
    beam[y] = rr / ratio;
    const int head = hk * ratio + (rr - beam[y] * ratio);
#pragma unroll
    for (int k = 0; k < QS; ++k) {
      const int d = F32 ? 16 * k + 4 * quad : 32 * k + 8 * quad;
      qf[y][k] = make_uint4(0, 0, 0, 0);
      if (d < D && r < R) qf[y][k] = *(const uint4*)(q + (size_t)(s0 + beam[y]) * q_ld + (size_t)head * D + d);
    }
  }
  const int n_b = lane < B ? max(0, min(n_raw, cap)) : 0, lo_b = window > 0 ? max(0, n_b - window) : 0;
  const uint64_t alive = __builtin_amdgcn_ballot_w64(n_b > 0);
  const int first_live = alive ? __builtin_ctzll(alive) : 0;
  // shared chunks: those that all beams have in shared pages, and all see from their first position on
  const int common = min(shared_g, wave_join(n_b > 0 ? n_b : 0x7fffffff, [](int a, int b) { return min(a, b); }));
  const int shared0 = alive ? (wave_join(lo_b, [](int a, int b) { return max(a, b); }) + CHUNK - 1) / CHUNK : 0;
  const int shared1 = alive ? max(shared0, common / CHUNK) : 0;
  // a beam's own chunks: from its first one on to its last, without the shared ones
  const int own0 = lo_b / CHUNK, own = lane >= b0 && lane <= b1 && n_b > 0 ? (n_b + CHUNK - 1) / CHUNK - own0 - (shared1 - shared0) : 0;
  const int own_to = wave_scan(own);
  const int n_shared = shared1 - shared0, items = n_shared + __builtin_amdgcn_readlane(own_to, DA_WAVE - 1);
  const int per = (items + splits - 1) / splits;
  const int item0 = z * per, item1 = min(items, item0 + per);
  const float scale2 = scale * 1.4426950408889634f;
  int len[RT], lo[RT];
  floatx4 acc[RT][DV];
  float m[RT], l[RT];
#pragma unroll
  for (int y = 0; y < RT; ++y) {
    const int n = __shfl(n_b, beam[y], DA_WAVE);
    lo[y] = __shfl(lo_b, beam[y], DA_WAVE);
    len[y] = r0 + TILE * y + col < R ? n : 0;
    m[y] = -INFINITY;
    l[y] = 0.f;
#pragma unroll
    for (int i = 0; i < DV; ++i) acc[y][i] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  const T* const kbase = cache + (size_t)hk * page * D;
  const T* const vbase = cache + (size_t)(Hkv + hk) * page * D;

  // Which chunk of whose table an item is (mine < 0: of all), and which of its positions are seen.
  struct Item {
    int mine, c0, first, last;
  };
  auto item_at = [&](int item) {
    Item it{-1, (shared0 + item) * CHUNK, 0, 0};
    it.first = it.c0;
    it.last = it.c0 + CHUNK - 1;
    if (item >= n_shared) {
      const int left = item - n_shared;
      it.mine = min((int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(own_to <= left)), b1);
      int chunk = __builtin_amdgcn_readlane(own0, it.mine) + left - (__builtin_amdgcn_readlane(own_to, it.mine) - __builtin_amdgcn_readlane(own, it.mine));
      if (chunk >= shared0) chunk += n_shared;
      it.c0 = chunk * CHUNK;
      it.first = max(it.c0, __builtin_amdgcn_readlane(lo_b, it.mine));
      it.last = min(it.c0 + CHUNK, __builtin_amdgcn_readlane(n_b, it.mine)) - 1;
    }
    return it;
  };
  // The pages of a lane's keys and values: keys (and groups of SPAN values) that nobody sees are read from a place that somebody does.
  constexpr int KI = F32 ? 4 : 2;                       // pages a lane has to look up: bfloat16: a group of 8 keys every 32
  struct Pages {
    int k[KI], v[KI];
  };
  auto pages_of = [&](const Item& it) {
    const int* bt = block_table + (size_t)(s0 + (it.mine < 0 ? first_live : it.mine)) * max_blocks;
    Pages p;
#pragma unroll
    for (int j = 0; j < KI; ++j) {
      const int kj = it.c0 + CHUNK / KI * j + (F32 ? col : 8 * (col / 4)), vj = it.c0 + CHUNK / KI * j + SPAN * quad;
      p.k[j] = bt[max(it.first, min(it.last, kj)) >> lg];
      p.v[j] = bt[max(it.first, min(it.last, vj)) >> lg];
    }
    return p;
  };

  Item now = item_at(min(item0 + wave, max(items - 1, 0)));
  Pages pages;
  if (item0 + wave < item1) pages = pages_of(now);
  for (int item = item0 + wave; item < item1; item += WAVES) {
    const int mine = now.mine, c0 = now.c0, first = now.first, last = now.last;
    const Pages here = pages;
    if (item + WAVES < item1) {                    // the next item's pages travel beside this one's keys and values
      now = item_at(item + WAVES);
      pages = pages_of(now);
    }
    auto step = [&](auto at_tag, auto cut_tag) {
      constexpr int AT = decltype(at_tag)::value;       // the step's place in the chunk
      constexpr bool CUT = decltype(cut_tag)::value;
      const int h0 = c0 + AT;
      if (CUT && (h0 > last || h0 + STEP <= first)) return;
      // ---- every load of the step, then the arithmetic
      uint4 kf[KP][QS], vf[VP][DV];
#pragma unroll
      for (int j = 0; j < KP; ++j) {
        const int key = h0 + (F32 ? 16 * j + col : 32 * (j / 2) + 8 * (col / 4) + 4 * (j % 2) + col % 4);
        // (a key that nobody sees: the one of its group's page that the page was looked up for)
        const int seen = CUT && (key < first || key > last) ? max(first, min(last, F32 ? key : key & ~7)) : key;
        const T* kp = kbase + (size_t)(uint32_t)max(here.k[(AT + 16 * j) / (CHUNK / KI)], 0) * page_elems + (size_t)(seen & pmask) * D;
#pragma unroll
        for (int k = 0; k < QS; ++k) {
          const int d = F32 ? 16 * k + 4 * quad : 32 * k + 8 * quad;
          // (a step that can lie past D: zeros, not a neighbour's numbers, of which zero times an infinite one is no number)
          if (2 * k + 2 <= QS && QS > 1) kf[j][k] = *(const uint4*)(kp + d);
          else {
            kf[j][k] = make_uint4(0, 0, 0, 0);
            if (d < D) kf[j][k] = *(const uint4*)(kp + d);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < VP; ++j) {
        const int k0 = h0 + 4 * SPAN * j + SPAN * quad;  // the lane's first key
        const int at = CUT ? max(first, min(last, k0)) & ~(SPAN - 1) : k0;
        const T* vp = vbase + (size_t)(uint32_t)max(here.v[(AT + 4 * SPAN * j) / (CHUNK / KI)], 0) * page_elems + (size_t)col * page + (at & pmask);
#pragma unroll
        for (int i = 0; i < DV; ++i) {
          vf[j][i] = *(const uint4*)vp;
          vp += 16 * (i + 1) < D ? 16 * page : 0;        // (a piece past D reads the last one again and is dropped)
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int y = 0; y < RT; ++y) {
        const bool takes = mine < 0 || mine == beam[y];
        floatx4 sc[KP];
#pragma unroll
        for (int j = 0; j < KP; ++j) sc[j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < QS; ++k)
#pragma unroll
          for (int j = 0; j < KP; ++j) {
            if (F32) {
              const uint32_t ka[4] = {kf[j][k].x, kf[j][k].y, kf[j][k].z, kf[j][k].w}, qa[4] = {qf[y][k].x, qf[y][k].y, qf[y][k].z, qf[y][k].w};
#pragma unroll
              for (int i = 0; i < 4; ++i)
                sc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ka[i]), __uint_as_float(qa[i]), sc[j], 0, 0, 0);
            } else {
              sc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kf[j][k]), __builtin_bit_cast(bf16x8_t, qf[y][k]), sc[j], 0, 0, 0);
            }
          }
        // ---- the lane's keys: four a piece, of column col's row
        float e[KP][4], top = -INFINITY;
#pragma unroll
        for (int j = 0; j < KP; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[j][i] = sc[j][i] * scale2;
            if (CUT) {
              const int key = h0 + (F32 ? 16 * j + 4 * quad + i : 32 * (j / 2) + 8 * quad + 4 * (j % 2) + i);
              e[j][i] = takes && key >= lo[y] && key < len[y] ? e[j][i] : -INFINITY;
            }
            top = fmaxf(top, e[j][i]);
          }
        const float m_new = fmaxf(m[y], quad_max(top)), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = exp_of_2(m[y] - m_use);
        m[y] = m_new;
        float add = 0.f;
#pragma unroll
        for (int j = 0; j < KP; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[j][i] = exp_of_2(e[j][i] - m_use);
            add += e[j][i];
          }
        l[y] = l[y] * alpha + add;
        uint4 part[3][VP];                              // bfloat16: the weights, 3 x 8 bits
        if (!F32) {
#pragma unroll
          for (int j = 0; j < VP; ++j) {
            uint32_t p4[3][4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              float x0 = e[2 * j + w / 2][2 * (w % 2)], x1 = e[2 * j + w / 2][2 * (w % 2) + 1];
#pragma unroll
              for (int p = 0; p < 3; ++p) {
                p4[p][w] = pack2_bf16(x0, x1);
                x0 -= __uint_as_float(p4[p][w] << 16);
                x1 -= __uint_as_float(p4[p][w] & 0xffff0000u);
              }
            }
#pragma unroll
            for (int p = 0; p < 3; ++p) part[p][j] = make_uint4(p4[p][0], p4[p][1], p4[p][2], p4[p][3]);
          }
        }
#pragma unroll
        for (int i = 0; i < DV; ++i) {
          floatx4 o;
#pragma unroll
          for (int x = 0; x < 4; ++x) o[x] = acc[y][i][x] * alpha;
#pragma unroll
          for (int j = 0; j < VP; ++j) {
            uint32_t v4[4] = {vf[j][i].x, vf[j][i].y, vf[j][i].z, vf[j][i].w};
            if (CUT) {                                  // positions that are not seen may hold anything
              const int k0 = h0 + 4 * SPAN * j + SPAN * quad;
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                if (F32) v4[w] = (k0 + w >= first && k0 + w <= last) ? v4[w] : 0u;
                else {
                  const int ka = k0 + 2 * w;
                  v4[w] &= ((ka >= first && ka <= last) ? 0x0000ffffu : 0u) | ((ka + 1 >= first && ka + 1 <= last) ? 0xffff0000u : 0u);
                }
              }
            }
            if (F32) {
#pragma unroll
              for (int x = 0; x < 4; ++x) o = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v4[x]), e[j][x], o, 0, 0, 0);
            } else {
              const uint4 v = make_uint4(v4[0], v4[1], v4[2], v4[3]);
#pragma unroll
              for (int p = 0; p < 3; ++p)
                o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v), __builtin_bit_cast(bf16x8_t, part[p][j]), o, 0, 0, 0);
            }
          }
          // (a column that takes no part keeps its sums: zero times another beam's infinite value is no number)
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[y][i][x] = !CUT || takes ? o[x] : acc[y][i][x];
        }
      }
    };
    auto all_steps = [&](auto cut_tag) {
      step(Int<0>{}, cut_tag);
      if constexpr (STEP < 64) step(Int<STEP>{}, cut_tag);
      if constexpr (STEP < 32) {
        step(Int<2 * STEP>{}, cut_tag);
        step(Int<3 * STEP>{}, cut_tag);
      }
    };
    if (mine < 0) all_steps(No{});
    else all_steps(Yes{});
  }

  // ---- the wavefronts' results joined
#pragma unroll
  for (int y = 0; y < RT; ++y) {
    l[y] += __shfl_xor(l[y], 16, DA_WAVE);
    l[y] += __shfl_xor(l[y], 32, DA_WAVE);
    const int row = TILE * y + col;
    if (quad == 0) {
      m_lds[wave][row] = len[y] > 0 ? m[y] : -INFINITY; // (a place without a beam went along in the shared chunks)
      l_lds[wave][row] = len[y] > 0 ? l[y] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < DV; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) acc_lds[wave][16 * i + 4 * quad + x][row] = len[y] > 0 ? acc[y][i][x] : 0.f;
  }
  __syncthreads();
  // 16 threads a row, 16 dimensions that follow each other (WAVES / 4 / RT rounds of all rows)
  static_assert(WAVES * DA_WAVE % (16 * ROWS) == 0, "whole rounds");
  const int row = t / 16 % ROWS, of_row = r0 + row;
  if (of_row >= R) return;
  float w[WAVES], mm = -INFINITY, ll = 0.f;
#pragma unroll
  for (int v = 0; v < WAVES; ++v) mm = fmaxf(mm, m_lds[v][row]);
  const float m_use = mm == -INFINITY ? 0.f : mm;
#pragma unroll
  for (int v = 0; v < WAVES; ++v) {
    w[v] = exp_of_2(m_lds[v][row] - m_use);
    ll += w[v] * l_lds[v][row];
  }
  const int bm = of_row / ratio, hd = hk * ratio + (of_row - bm * ratio);
  const float inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
  T* o_row = out + (size_t)(s0 + bm) * out_ld + (size_t)hd * D;
  float* p_row = partial + (((size_t)(s0 + bm) * Hq + hd) * splits + z) * (D + 2);
#pragma unroll
  for (int k = 0; k < DMAX; k += WAVES * DA_WAVE / ROWS) {
    const int d = k + t / (16 * ROWS) * 16 + t % 16;
    if (d >= D) break;
    float o = 0.f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) o += w[v] * acc_lds[v][d][row];
    if (splits == 1) from_f32(o_row + d, o * inv);
    else p_row[d] = o;
  }
  if (splits > 1 && t < 16 * ROWS && t % 16 == 0) {
    p_row[D] = mm;
    p_row[D + 1] = ll;
  }
}

// A wavefront a (sequence, head): a share a lane for the maxima and sums, then a dimension a lane.
#define MERGE_WAVES 4
template <typename T>
__global__ void __launch_bounds__(MERGE_WAVES * DA_WAVE)
attn_beams_merge_kernel(const float* __restrict__ partial, int splits, int pairs, int Hq, int D, T* __restrict__ out, int out_ld) {
  const int lane = threadIdx.x % DA_WAVE, pair = blockIdx.x * MERGE_WAVES + threadIdx.x / DA_WAVE;
  if (pair >= pairs) return;
  const int s = pair / Hq, h = pair - s * Hq;
  const float* p = partial + (size_t)pair * splits * (D + 2);
  const float* mine = p + (size_t)(lane < splits ? lane : 0) * (D + 2) + D;
  const float m = lane < splits ? mine[0] : -INFINITY, l = lane < splits ? mine[1] : 0.f;
  auto load = [&](float v[8], int d0, int z0) {
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = p[(size_t)min(z0 + u, splits - 1) * (D + 2) + min(d0 + lane, D - 1)];
  };
  float v[8];
  load(v, 0, 0);                                        // (the first of them travel beside the maxima)
  const float mm = wave_max(m), m_use = mm == -INFINITY ? 0.f : mm;
  const float w = lane < splits ? exp_of_2(m - m_use) : 0.f;
  const float ll = wave_sum(w * l), inv = ll > 0.f || ll != ll ? 1.f / ll : 0.f;
  for (int d0 = 0; d0 < D; d0 += DA_WAVE) {
    float o = 0.f;
    for (int z0 = 0; z0 < splits; z0 += 8) {
      if (d0 + z0 > 0) load(v, d0, z0);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float wz = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), min(z0 + u, DA_WAVE - 1)));
        o += z0 + u < splits ? wz * v[u] : 0.f;
      }
    }
    if (d0 + lane < D) from_f32(out + (size_t)s * out_ld + (size_t)h * D + d0 + lane, o * inv);
  }
}

extern "C" int da_attn_beams_takes(int D, int page) {
  return D % 16 == 0 && D >= 16 && D <= BEAMS_MAX_D && page >= 16 && (page & (page - 1)) == 0;
}

// Rows of a workgroup.  Two tiles where with one there would be more than a workgroup a compute unit, all of which read what they share: 10 x 5 beams,
// 68 / 17 heads of 64, 853 positions 21.4 us for 27.7, 7 x 7 beams, 95 / 19 heads, 1,956 positions 40.4 for 49.4; with fewer workgroups the
// second tile's arithmetic is what is waited for (13 x 4 beams, 15 / 3 heads of 80, 3,365 positions 29.8 for 24.8).  Above 64 the registers do not hold it.
static long beam_groups(int G, int B, int Hq, int Hkv, int rows) { return (long)G * Hkv * da_ceil_div((long)B * (Hq / Hkv), rows); }
static int beam_rows(int G, int B, int Hq, int Hkv, int D) {
  return (long)B * (Hq / Hkv) > TILE && D <= 64 && beam_groups(G, B, Hq, Hkv, TILE) > 256 ? 2 * TILE : TILE;
}

// How many workgroups share a group's positions: from the step's shape only.  One workgroup a compute unit; a second kernel, which joins the shares,
// does not pay for few chunks (bfloat16, 1 x 4 beams of 12 heads of 64, 9 chunks: 7.7 us with one workgroup, 8.1 with four, and a launch more on the
// host; 16 chunks 9.8 and 8.0; heads of 128, 11 chunks 13.8 and 10.3).  In 32-bit, whose products take 16 times as long, it does: 2 x 5 beams, 9 chunks 19.3 and 11.8.
extern "C" int da_attn_beams_splits(int G, int B, int Hq, int Hkv, int D, int dtype, int max_blocks, int page) {
  if (G <= 0 || B <= 0 || Hkv <= 0 || Hq < Hkv || max_blocks <= 0 || page <= 0) return 1;
  const long groups = beam_groups(G, B, Hq, Hkv, beam_rows(G, B, Hq, Hkv, D));
  const long chunks = ((long)max_blocks * page + CHUNK - 1) / CHUNK;
  long n = chunks < (dtype == DA_F32 ? 4 : (D <= 64 ? 12 : 8)) ? 1 : 256 / groups;
  if (n > chunks / 2) n = chunks / 2;
  return n < 1 ? 1 : (n > DA_WAVE ? DA_WAVE : (int)n);
}

// Wavefronts of a workgroup.  8 where there is one workgroup a compute unit, which they fill by themselves (us a call in a chain, 8 / 4): 8 x 8 beams of 25 heads
// over 1,003 positions 18.1 / 21.1, 1 x 4 of 12 heads over 531 8.0 / 9.1, 24 beams of 7 heads over 3,456 11.7 / 11.9.  4 where more share one, and where each has so
// many chunks that 4 wavefronts keep the memory busy: 4 x 4 beams of 32 / 8 heads of 128 over 32,701 positions, 64 chunks each, 116 / 108.  26 chunks
// each lie between: heads of 64 29.0 / 30.4, 26.7 / 28.9, 25.7 / 27.0, of 128 53.9 / 52.4, 68.6 / 71.6.
static int beam_waves(long groups, int splits, int max_blocks, int page) {
  return groups * splits > 256 || (long)max_blocks * page / CHUNK >= 48L * splits ? 4 : 8;
}

// Whether a step of beams is ahead here or in the kernels that take a sequence by itself (bfloat16 attn_decode.hip, 32-bit attn_f32.hip): both sides' times,
// us, from the step's shape and what its sequences see.  A start; what joining shares adds; then the larger of the workgroups' chains (rounds of 64 or 32
// keys a wavefront, and one for the way in and out) where compute units take several in turn, and the bytes that are asked for (here those of shared keys
// once a workgroup; much of it comes from caches).  The numbers are fitted to 20,584 measured pairs: 2 to 32 beams, 1 to 16 groups, 2 to 32 heads of 16 to 256, 1 to 8 of
// them a key head, 11 to 32,000 positions in tables up to 32,768 wide, windows from 64.  Of those the choice is the faster kernel or within 5 % of it in 92 of 100, 1.3 % behind it on
// average, 1.84 times at the worst (one by the table's width alone: 60 of 100, 18 %, 14.5 times).  us, the others / here: bfloat16, 2 x 3 beams of 4 heads of 16 in a
// table of 2,048 positions: 23 positions 6.5 / 7.5, 547 7.7 / 7.6; 4 x 32 of 25 heads of 64, 393 37.8 / 23.3; 1 x 3 of 32 / 8 heads of 128, 102 5.0 / 9.4; 8 x 5 of 8 / 1
// heads of 64, 23 in 4,096 4.7 / 9.0; 1 x 4 of 12 heads of 64, 531 5.4 / 7.8, 4,000 12.1 / 9.3; 32-bit: 1 x 4 of 2 heads of 48, 33 5.1 / 10.4; 1 x 8 of 8 heads of 128, a window of 64 7.9 / 14.8;
// 1 x 3 of 12 heads of 64, 3,989 68.9 / 17.7.
struct StepTime {
  float units, units_wide;       // of a compute unit, that a workgroup takes: head sizes up to 64, above
  float start, start_d;          // _d: for each 64 of the head size
  float join, join_share;
  float round, round_d;
  float megabyte;
};
static float step_us(const StepTime& t, int D, int d, int shares, float workgroups, float rounds, float megabytes) {
  const float in_turn = workgroups / 256 * (d <= 64 ? t.units : t.units_wide), d64 = d / 64.f;
  const float chain = (in_turn > 1 ? in_turn : 1) * (rounds + 1) * (t.round + t.round_d * d64), bytes = megabytes * t.megabyte;
  return t.start + t.start_d * d64 + (shares > 1 ? t.join + t.join_share * shares * da_ceil_div(D, 64) : 0) + (chain > bytes ? chain : bytes);
}

// By how many nanoseconds a step is ahead here (negative: behind; where the two are within 6 % it stays here, where nothing is read twice).  visible:
// positions that a sequence sees, shared: those of them that its group shares, both on average; decode_splits: shares of the other kernel (bfloat16).
extern "C" int da_attn_beams_ahead_ns(int G, int B, int Hq, int Hkv, int D, int dtype, int max_blocks, int page, int splits, int decode_splits,
                                      int visible, int shared) {
  if (G <= 0 || B <= 0 || Hkv <= 0 || Hq < Hkv || max_blocks <= 0 || splits <= 0 || decode_splits <= 0 || visible <= 0 || !da_attn_beams_takes(D, page)) return -1;
  static const StepTime decode_bf16 = {0.69f, 1.43f, 1.97f, 0.403f, 2.36f, 0.189f, 1.71f, 0.305f, 0.112f};
  static const StepTime decode_f32 = {0.72f, 0.956f, 1.36f, 0.f, 0.f, 0.f, 2.06f, 1.96f, 0.146f};
  static const StepTime beams_bf16 = {0.909f, 0.817f, 2.08f, 0.044f, 2.56f, 0.0617f, 1.52f, 1.05f, 0.204f};
  static const StepTime beams_f32 = {0.891f, 0.686f, 0.f, 0.f, 3.52f, 0.0611f, 2.31f, 3.38f, 0.221f};
  const bool f32 = dtype == DA_F32;
  const float S = (float)G * B, v = visible, s = shared < visible ? (shared > 0 ? shared : 0) : visible, key_mb = 2.f * D * (f32 ? 4 : 2) * 1e-6f;
  // the others: a workgroup a (sequence, head, share); shares are by the table's width, so that a short context lies in the first
  float span = 1e9f, a_wave = 32.f * 8;
  if (!f32) {
    span = (float)((((long)max_blocks * page + decode_splits - 1) / decode_splits + CHUNK - 1) / CHUNK * CHUNK);
    a_wave = (float)CHUNK * (S * Hq * decode_splits <= 256 && D <= 64 ? 16 : 8);
  }
  const float with_keys = v / span < 1 ? 1 : (v / span > decode_splits ? decode_splits : v / span);
  const float others = step_us(f32 ? decode_f32 : decode_bf16, D, D, f32 ? 1 : decode_splits, S * Hq * (f32 ? 1 : with_keys), (v < span ? v : span) / a_wave, S * Hq * v * key_mb);
  // here: the shared chunks and those of the beams whose rows a workgroup has, whole ones
  const int rows = beam_rows(G, B, Hq, Hkv, D), ratio = Hq / Hkv;
  const float groups = (float)beam_groups(G, B, Hq, Hkv, rows), beams = rows < B * ratio ? (float)rows / ratio : (float)B;
  const float chunks = s / CHUNK + beams * ((v - s) / CHUNK + 0.75f);
  const float once = G * (s + B * (v - s)) * Hkv, asked = 0.8f * groups * (s + beams * (v - s));
  const int waves = D > 128 ? 4 : (rows > TILE ? 8 : beam_waves((long)groups, splits, max_blocks, page));
  const float joined_mb = splits > 1 ? S * Hq * splits * D * 8e-6f : 0.f;
  const float here = step_us(f32 ? beams_f32 : beams_bf16, D, D <= 32 ? 32 : (D <= 64 ? 64 : (D <= 128 ? 128 : 256)), splits, groups * splits,
                             chunks / splits / waves, (once > asked ? once : asked) * key_mb) + joined_mb * (f32 ? 0.482f : 0.381f);
  const float ns = (1.06f * others - here) * 1000;
  return ns > 1e9f ? 1000000000 : (ns < -1e9f ? -1000000000 : (int)ns);
}

template <typename T, int DK, int STEP>
static void beams_launch(hipStream_t s, const void* q, int q_ld, const void* cache, const int* block_table, int max_blocks, const int* seq_lens,
                         const int* shared, int G, int B, int Hq, int Hkv, int D, int page, float scale, int window, void* out, int out_ld,
                         int splits, float* partial) {
  const int rows = beam_rows(G, B, Hq, Hkv, D);
  const dim3 grid(Hkv * da_ceil_div((long)B * (Hq / Hkv), rows), G, splits);
  const int waves = beam_waves(beam_groups(G, B, Hq, Hkv, rows), splits, max_blocks, page);
#define DA_BEAMS_AS(WAVES, RT) \
  hipLaunchKernelGGL((attn_beams_kernel<T, DK, STEP, WAVES, RT>), grid, dim3(WAVES * DA_WAVE), 0, s, (const T*)q, q_ld, (const T*)cache, block_table, \
                     max_blocks, seq_lens, shared, B, Hq, Hkv, D, page, scale, window, (T*)out, out_ld, splits, partial)
  if constexpr (DK == 8) {                              // (registers for 4 wavefronts only)
    DA_BEAMS_AS(4, 1);
  } else {
    if constexpr (DK <= 2) {
      if (rows > TILE) {
        DA_BEAMS_AS(8, 2);
        return;
      }
    }
    if (waves == 8) DA_BEAMS_AS(8, 1);
    else DA_BEAMS_AS(4, 1);
  }
#undef DA_BEAMS_AS
}

extern "C" int da_attn_beams(const void* q, int q_ld, const void* cache, int dtype, const int* block_table, int max_blocks, const int* seq_lens,
                             const int* shared, int G, int B, int Hq, int Hkv, int D, int page, float scale, int window, void* out, int out_ld,
                             int splits, float* workspace, long workspace_floats, void* stream) {
  DA_REQUIRE(G >= 0 && B > 0 && B <= BEAMS_MAX && (long)G * B <= 65535 && Hkv > 0 && Hq > 0 && Hq <= 32767 && Hq % Hkv == 0 && max_blocks > 0 && window >= 0,
             "attention_beams: bad sizes (groups=%d beams=%d heads=%d/%d blocks=%d window=%d; at most %d beams)", G, B, Hq, Hkv, max_blocks, window, BEAMS_MAX);
  DA_REQUIRE(da_attn_beams_takes(D, page), "attention_beams: head size %d (multiples of 16 up to %d), page %d (powers of two from 16)", D, BEAMS_MAX_D, page);
  DA_REQUIRE(dtype == DA_F32 || dtype == DA_BF16, "attention_beams: dtype %d", dtype);
  const int el = dtype == DA_F32 ? 4 : 2;
  DA_REQUIRE((uintptr_t)q % 16 == 0 && (long)q_ld * el % 16 == 0 && (uintptr_t)cache % 16 == 0, "attention_beams: q and the cache must lie on 16 bytes");
  DA_REQUIRE((long)max_blocks * page <= 0x7fffff00L && 2L * Hkv * page * D <= 0x7fffffffL, "attention_beams: a page or a table is too large");
  DA_REQUIRE(splits >= 1 && splits <= DA_WAVE, "attention_beams: %d shares (1 to 64)", splits);
  const long need = splits > 1 ? (long)G * B * Hq * splits * (D + 2) : 0;
  DA_REQUIRE(need == 0 || (workspace && workspace_floats >= need), "attention_beams: %ld floats of workspace are needed, found %ld", need, workspace_floats);
  if (G == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
#define DA_BEAMS(T, DK, STEP) beams_launch<T, DK, STEP>(s, q, q_ld, cache, block_table, max_blocks, seq_lens, shared, G, B, Hq, Hkv, D, page, scale, window, out, out_ld, splits, workspace)
  if (dtype == DA_F32) {
    if (D <= 32) DA_BEAMS(float, 1, 32);
    else if (D <= 64) DA_BEAMS(float, 2, 32);
    else if (D <= 128) DA_BEAMS(float, 4, 16);
    else DA_BEAMS(float, 8, 16);
  } else {
    if (D <= 32) DA_BEAMS(bf16_t, 1, 64);
    else if (D <= 64) DA_BEAMS(bf16_t, 2, 64);
    else if (D <= 128) DA_BEAMS(bf16_t, 4, 32);
    else DA_BEAMS(bf16_t, 8, 32);
  }
#undef DA_BEAMS
  DA_CHECK_LAUNCH("attention_beams");
  if (splits > 1) {
    const int pairs = G * B * Hq;
    const dim3 grid(da_ceil_div(pairs, MERGE_WAVES)), block(MERGE_WAVES * DA_WAVE);
    if (dtype == DA_F32) hipLaunchKernelGGL((attn_beams_merge_kernel<float>), grid, block, 0, s, workspace, splits, pairs, Hq, D, (float*)out, out_ld);
    else hipLaunchKernelGGL((attn_beams_merge_kernel<bf16_t>), grid, block, 0, s, workspace, splits, pairs, Hq, D, (bf16_t*)out, out_ld);
    DA_CHECK_LAUNCH("attention_beams (merge)");
  }
  return 0;
}
