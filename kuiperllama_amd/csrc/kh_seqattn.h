// kh_seqattn.h — causal attention of many sequences' tokens over keys that lie in rows (whole prompts) or in pages of a cache.
//
// With s_j = scale q . k_j over the keys that a query sees:  m = max s_j,  l = sum exp(s_j - m),  out = sum exp(s_j - m) v_j / l,
// in one pass over the keys with a running m, l and output.
//
// Query rows.  The heads that share a key head are rows of one product: row r of a sequence is its token r / G and head r % G of the
// group, G = heads / kv_heads, so 32 rows are 32 tokens of one head each or 8 tokens of a group of four.  A wave takes 32 rows.
// S^T = K Q^T on 32 x 32 tiles: a lane ends with the scores of ONE query (its column) and 16 of a tile's 32 keys, rows
// 8 (i / 4) + 4 h + i % 4 for lane half h.  So the running maximum and sum are lane scalars and one swap of halves, and as the order
// of a sum is free, the weights are the second operand of O^T = V^T P^T as they are: the first operand just takes its keys
// in the same order, out of V's rows in LDS by the transposing read (bf16) or an element at a time (fp32).
//
// Exponentials run in base two: p = 2^(c s - c m), c = scale log2(e), one fma a score.  m follows the running maximum only when
// a score passes it by 8 / c: weights then stay below 2^8, which fp32 sums and products in bf16 hold as well as those below one,
// and most tiles spare the output its factor.
// Roundings: scores, weights, sums and outputs are fp32; for bf16 the weights are rounded to bf16 for their product with the
// values (the sum l takes them unrounded).
#pragma once
#include "kh_lgemm.h"

namespace khm {
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// 32 x 32 products of 32-byte k-blocks.  A fragment is 16 bytes a lane: row l & 31, bytes [16 (l / 32), + 16) of the block.
template <class T>
struct Tile32;
template <>
struct Tile32<bf16> {
  typedef bf16x8 frag;
  static __device__ __forceinline__ f32x16 mma(const frag& a, const frag& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Tile32<float> {
  typedef f32x4 frag;
  static __device__ __forceinline__ f32x16 mma(const frag& a, const frag& b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

// Where keys and values are.  Strides in bytes.
struct SeqKv {
  const char *k, *v;
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
  const int32_t* pages;  // nullptr: rows, those of the sequence's tokens
  int64_t table_stride;
  int n_pages, page_size, most;  // most: places of a sequence's row of the table
  uint32_t magic;  // place / page_size = umulhi(place, magic) >> shift; 0: page_size 1
  int shift;
  const int32_t* lengths;
};
struct SeqArgs {
  SeqKv kv;
  const char* q;
  char* out;
  int64_t q_token, q_head, o_token, o_head;  // bytes
  const int32_t* offsets;
  int n_tokens, n_seqs, heads, kv_heads, group, kchunks, vchunks, window;  // chunks of 16 bytes of a row
  float c;                                                                 // scale log2(e)
};

// 16 bytes of zeros, for the chunks of a tile behind the end of its rows
__device__ const f32x4 seq_zeros = {0.f, 0.f, 0.f, 0.f};

// One sequence, with what the device's own numbers may not do to memory cut off.
struct SeqSpan {
  int first, n, length;  // tokens [first, first + n), keys
  bool bad;              // more keys than the table has places for
};
__device__ __forceinline__ SeqSpan seq_span(const SeqArgs& a, int b) {
  SeqSpan s;
  const int lo = a.offsets[b], hi = a.offsets[b + 1];
  s.first = lo < 0 ? 0 : (lo > a.n_tokens ? a.n_tokens : lo);
  const int end = hi > a.n_tokens ? a.n_tokens : hi;
  s.n = end > s.first ? end - s.first : 0;
  s.length = a.kv.lengths ? a.kv.lengths[b] : s.n;
  s.bad = a.kv.lengths && s.length > a.kv.most;
  if (s.bad) s.length = a.kv.most;
  if (s.length < 0) s.length = 0;
  return s;
}

template <class T, int DP>
struct SeqCfg {
  static constexpr int E = 16 / (int)sizeof(T);
  static constexpr int RB = DP * (int)sizeof(T);  // bytes of a staged row
  static constexpr int CB = RB / 16;              // its chunks
  static constexpr int NKB = RB / 32;             // its 32-byte k-blocks
  static constexpr int NMB = DP / 32;             // 32-column blocks of the output
  static constexpr bool TIGHT = RB > 256;         // queries and outputs fill the registers: reads of LDS stay near their use
  static constexpr bool HOLD = RB <= 512;         // queries in registers; else read again for each tile, under 128 products of 64 cycles
  // LDS: chunk c of row r lies in slot c ^ turn(r).  Reads of a column of chunks over rows (keys), and of 32 bytes of four and
  // four rows (values), then touch every bank once.  turn(r + 8) = turn(r), and turn(4 + i) = turn(4) ^ turn(i): a lane's addresses of a
  // tile are one of its own, turned by constants.
  static __device__ __forceinline__ int turn(int r) { return RB == 128 ? ((r >> 1) & 3) * 2 : (r & 7) * 2; }
};

template <class X>
__device__ __forceinline__ X lds_read(unsigned addr) {
  return *(const __attribute__((address_space(3))) X*)(size_t)addr;
}

// The running state of 32 query rows, a lane's row being l & 31.
template <class T, int DP>
struct SeqState {
  typedef SeqCfg<T, DP> C;
  typedef typename Tile32<T>::frag frag;
  frag q[C::HOLD ? C::NKB : 1];
  const char* row;  // of the queries
  int chunks;
  f32x16 o[C::NMB];
  float m, l;  // l: this half's keys

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < C::NMB; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[n][i] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }
  __device__ __forceinline__ frag query(int b, int half) const {
    frag f;
    const int c = 2 * b + half;
    if (c < chunks) f = *(const frag*)(row + 16 * c);
    else
#pragma unroll
      for (int i = 0; i < C::E; ++i) f[i] = (T)0.f;
    return f;
  }
  __device__ __forceinline__ void load_q(const char* at, int half, int n) {
    row = at;
    chunks = n;
    if constexpr (C::HOLD)
#pragma unroll
      for (int b = 0; b < C::NKB; ++b) q[b] = query(b, half);
  }
  // scores of 32 keys, rows r0 .. of the tile at K
  __device__ __forceinline__ f32x16 scores(unsigned K, int r0, int lane) const {
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
    const int r = lane & 31;
    const unsigned at = K + (unsigned)(r * C::RB + 16 * ((lane >> 5) ^ C::turn(r)));
#pragma unroll
    for (int b = 0; b < C::NKB; ++b) {
      s = Tile32<T>::mma(lds_read<frag>((at ^ (32 * b)) + r0 * C::RB), C::HOLD ? q[C::HOLD ? b : 0] : query(b, lane >> 5), s);
      if (C::TIGHT && b % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
    return s;
  }
  // the new maximum, and the factor of what there was
  __device__ __forceinline__ void follow(float mx, float c) {
    if (__builtin_amdgcn_ballot_w64(mx > m + 8.f / c || (m == -INFINITY && mx > m)) != 0) {
      const float to = fmaxf(m, mx), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - to) * c);
      m = to;
      l *= f;
#pragma unroll
      for (int n = 0; n < C::NMB; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[n][i] *= f;
    }
  }
  __device__ __forceinline__ f32x16 weigh(const f32x16& s, float c) {
    const float base = m == -INFINITY ? 0.f : -m * c;  // no key seen yet: 2^-inf
    f32x16 p;
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, base));
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += p[i];
    l += t;
    return p;
  }
  // O^T += V^T P^T for 32 keys, rows r0 .. of the tile at V
  __device__ __forceinline__ void add(const f32x16& p, unsigned V, int r0, int lane) {
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      const int r = 4 * half + ((lane >> 2) & 3);  // of eight
      const unsigned at = V + (unsigned)(r * C::RB + 16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ C::turn(r)) + 8 * (lane & 1));
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        bf16x8 b;
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = (bf16)p[8 * t + i];
#pragma unroll
        for (int n = 0; n < C::NMB; ++n) {
          bf16x8 a;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const bf16x4 v = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(size_t)((at ^ (64 * n)) + (r0 + 16 * t + 8 * g) * C::RB)));
#pragma unroll
            for (int i = 0; i < 4; ++i) a[4 * g + i] = v[i];
          }
          o[n] = Tile32<T>::mma(a, b, o[n]);
          if (C::TIGHT && n % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        }
      }
    } else {
      const unsigned at = V + (unsigned)(4 * half * C::RB + 16 * (((lane & 31) >> 2) ^ C::turn(4 * half)) + 4 * (lane & 3));
#pragma unroll
      for (int i = 0; i < 16; ++i) {
#pragma unroll
        for (int n = 0; n < C::NMB; ++n)
          o[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(lds_read<float>((at ^ (16 * C::turn(i & 3) + 128 * n)) + (r0 + 8 * (i >> 2) + (i & 3)) * C::RB), p[i], o[n],
                                                      0, 0, 0);
        if (C::TIGHT) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  // does any output hold what is no number
  __device__ __forceinline__ bool odd() const {
    float s = 0.f;  // x - x is 0 for numbers, NaN for the others
#pragma unroll
    for (int n = 0; n < C::NMB; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) s += o[n][i] - o[n][i];
    return !(s == 0.f);
  }
};

// ---- staging ---------------------------------------------------------------------------------------------------------------------
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 64 lanes x 16 B, every lane from an address of its own, to LDS [dst + 16 * lane]
__device__ __forceinline__ void dma_x4_from(const char* addr, unsigned dst) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(addr), "s"(dst) : "memory", "m0");
}
#pragma clang diagnostic pop

// Keys [lo, hi) of a sequence are those that anyone of a workgroup's rows sees: no other row, and no other page, is touched.
struct SeqKeys {
  const char *k, *v;  // of the key head; of the sequence's first token where keys are rows
  const int32_t* table;
  int lo, hi;
  bool bad;  // a page outside the cache was named, or the table is too short
};
__device__ __forceinline__ SeqKeys seq_keys(const SeqArgs& a, int b, int head, const SeqSpan& s, int first_place, int last_place) {
  SeqKeys x;
  x.k = a.kv.k + head * a.kv.k_head;
  x.v = a.kv.v + head * a.kv.v_head;
  x.table = nullptr;
  if (a.kv.pages) {
    x.table = a.kv.pages + b * a.kv.table_stride;
  } else {
    x.k += s.first * a.kv.k_slot;
    x.v += s.first * a.kv.v_slot;
  }
  x.lo = a.window > 0 && first_place >= a.window ? first_place - a.window + 1 : 0;
  x.hi = last_place + 1;
  x.bad = s.bad;
  return x;
}
// Bytes from x.k and x.v to the row of a key.
template <bool PAGED>
__device__ __forceinline__ void seq_row(const SeqArgs& a, SeqKeys& x, int place, int64_t& ko, int64_t& vo) {
  if constexpr (PAGED) {
    const int p = a.kv.magic ? (int)(__umulhi((uint32_t)place, a.kv.magic) >> a.kv.shift) : place;
    const int slot = place - p * a.kv.page_size;
    int page = x.table[p];
    if ((unsigned)page >= (unsigned)a.kv.n_pages) {
      page = 0;
      x.bad = true;
    }
    ko = page * a.kv.k_page + slot * a.kv.k_slot;
    vo = page * a.kv.v_page + slot * a.kv.v_slot;
  } else {
    ko = place * a.kv.k_slot;
    vo = place * a.kv.v_slot;
  }
}
// One of WAVES waves brings its part of keys k0 .. k0 + BN - 1 and their values to LDS.
template <class T, int DP, int BN, int WAVES, bool PAGED>
__device__ __forceinline__ void seq_stage(const SeqArgs& a, SeqKeys& x, int k0, unsigned K, unsigned V, int wave, int lane) {
  typedef SeqCfg<T, DP> C;
  constexpr int NL = BN * C::CB / (64 * WAVES);
  static_assert(NL * 64 * WAVES == BN * C::CB, "whole requests");
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const int i = (WAVES * j + wave) * 64 + lane, r = i / C::CB, c = (i - r * C::CB) ^ C::turn(r);
    int place = k0 + r;
    place = place < x.lo ? x.lo : (place >= x.hi ? x.hi - 1 : place);
    int64_t ko, vo;
    seq_row<PAGED>(a, x, place, ko, vo);
    const unsigned at = (unsigned)((WAVES * j + wave) * 1024);
    dma_x4_from(c < a.kchunks ? x.k + ko + 16 * c : (const char*)&seq_zeros, K + at);
    dma_x4_from(c < a.vchunks ? x.v + vo + 16 * c : (const char*)&seq_zeros, V + at);
    if (C::TIGHT) __builtin_amdgcn_sched_barrier(0);
  }
}

// One query by one wave from global memory, 64 keys at a time: a lane has a key for the scores, four columns for the output.  A key
// that the query does not see is not touched, so that what it holds cannot reach it (in a product over a tile it is zero times
// the value, which is no zero for what is no number): for the rows where that seems to have happened.
template <class T, bool PAGED>
__device__ __forceinline__ void seq_one(const SeqArgs& a, SeqKeys& x, const char* q, char* out, int place, int lane) {
  typedef typename Tile<T>::frag frag;
  constexpr int E = Tile<T>::N;
  const int lo = a.window > 0 && place >= a.window ? place - a.window + 1 : 0, cols = a.vchunks * E;
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = lo; k0 <= place; k0 += 64) {
    const int key = k0 + lane;
    int64_t ko = 0, vo = 0;
    float s = -INFINITY;
    if (key <= place) {
      seq_row<PAGED>(a, x, key, ko, vo);
      s = 0.f;
      for (int c = 0; c < a.kchunks; ++c) {
        const frag u = *(const frag*)(q + 16 * c), w = *(const frag*)(x.k + ko + 16 * c);
        for (int i = 0; i < E; ++i) s = __builtin_fmaf((float)u[i], (float)w[i], s);
      }
    }
    const float to = fmaxf(m, wave_max(s)), base = to == -INFINITY ? 0.f : -to * a.c;
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - to) * a.c), p = __builtin_amdgcn_exp2f(__builtin_fmaf(s, a.c, base));
    m = to;
    l = l * f + wave_sum(p);
    for (int i = 0; i < 4; ++i) o[i] *= f;
    const int n = place - k0 < 63 ? place - k0 + 1 : 64;
    for (int j = 0; j < n; ++j) {
      const float w = __shfl(p, j);
      const char* row = x.v + __shfl((long long)vo, j);
      for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < cols && w != 0.f) o[i] = __builtin_fmaf(w, (float)((const T*)row)[lane + 64 * i], o[i]);
    }
  }
  const float f = __builtin_amdgcn_ballot_w64(x.bad) ? NAN : (l == 0.f ? 0.f : 1.0f / l);
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < cols) ((T*)out)[lane + 64 * i] = (T)(o[i] * f);
}

// The sequence whose slots hold slot i, where sequence b has the slots from offsets[b] G / BM + b on: at least as many as it has
// tiles of BM rows, as floor((x + y) / BM) + 1 - floor(x / BM) >= ceil(y / BM).  64 candidates a trip.
__device__ __forceinline__ int seq_slot_base(const SeqArgs& a, int b, int rows) {
  const int o = a.offsets[b];
  return (int)((int64_t)(o < 0 ? 0 : (o > a.n_tokens ? a.n_tokens : o)) * a.group / rows) + b;
}
__device__ __forceinline__ int seq_of_slot(const SeqArgs& a, int i, int rows, int lane) {
  int lo = 0, n = a.n_seqs;
  while (n > 1) {
    const int step = (n + 63) / 64, b = lane * step;
    const bool at = b < n && seq_slot_base(a, lo + b, rows) <= i;
    const uint64_t yes = __builtin_amdgcn_ballot_w64(at);
    const int k = yes ? 63 - __builtin_clzll(yes) : 0;
    lo += k * step;
    n = n - k * step < step ? n - k * step : step;
  }
  return lo;
}

template <class T, int DP>
struct SeqTiles {
  static constexpr int W = 4, BM = 32 * W;
  static constexpr int BN = sizeof(T) == 2 ? 64 : 32;
  static constexpr int TB = BN * SeqCfg<T, DP>::RB;  // bytes of a tile of keys
  static constexpr int LDS = 4 * TB;                 // two tiles of keys and values each
};

// Four waves of 32 rows each share the tiles of keys and values.  grid (slots * kv_heads): the key heads side by side, so that a
// key head's tiles stay with one XCD's L2 where their number is a multiple of eight.  Long tiles of a sequence first.
template <class T, int DP, bool PAGED>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void k_seq_tiles(const SeqArgs a) {
  typedef SeqTiles<T, DP> S;
  typedef SeqCfg<T, DP> C;
  extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = (int)blockIdx.x % a.kv_heads, slot = (int)blockIdx.x / a.kv_heads;
  const int b = __builtin_amdgcn_readfirstlane(seq_of_slot(a, slot, S::BM, lane));
  const SeqSpan sp = seq_span(a, b);
  const int rows = sp.n * a.group;
  const int tiles = (rows + S::BM - 1) / S::BM, tile = tiles - 1 - (slot - seq_slot_base(a, b, S::BM));
  if (tile < 0 || tile >= tiles) return;
  auto place_of = [&](int r) __attribute__((always_inline)) { return sp.length - sp.n + (r < rows ? r : rows - 1) / a.group; };
  const int r0 = tile * S::BM, w0 = r0 + 32 * wave, row = w0 + (lane & 31);
  SeqKeys x = seq_keys(a, b, head, sp, place_of(r0), place_of(r0 + S::BM - 1));
  const int w_first = place_of(w0), w_last = place_of(w0 + 31), place = place_of(row);
  const int token = (row < rows ? row : rows - 1) / a.group, h = head * a.group + (row < rows ? row : rows - 1) - token * a.group;
  SeqState<T, DP> st;
  st.load_q(a.q + (sp.first + token) * a.q_token + h * a.q_head, half, a.kchunks);
  const unsigned lds0 = (unsigned)__builtin_amdgcn_readfirstlane((int)kh_lds_addr(smem_raw));
  const int t_lo = x.lo / S::BN, t_hi = (x.hi + S::BN - 1) / S::BN;
  auto issue = [&](int t) __attribute__((always_inline)) {
    const unsigned at = lds0 + (unsigned)((t & 1) * 2 * S::TB);
    seq_stage<T, DP, S::BN, S::W, PAGED>(a, x, t * S::BN, at, at + S::TB, wave, lane);
  };
  char* out = a.out + (sp.first + token) * a.o_token + h * a.o_head;
  st.clear();
  if (t_lo < t_hi) issue(t_lo);
  for (int t = t_lo; t < t_hi; ++t) {
    wait_vm<0>();     // this tile has landed
    __syncthreads();  // for every wave, and everyone is done with the tile before
    if (t + 1 < t_hi) issue(t + 1);
    const int k0 = t * S::BN;
    if (k0 > w_last || (a.window > 0 && k0 + S::BN - 1 <= w_first - a.window)) continue;  // nothing that this wave sees
    const unsigned K = lds0 + (unsigned)((t & 1) * 2 * S::TB), V = K + S::TB;
    f32x16 s[S::BN / 32];
#pragma unroll
    for (int n = 0; n < S::BN / 32; ++n) s[n] = st.scores(K, 32 * n, lane);
    if (k0 + S::BN - 1 > w_first || (a.window > 0 && k0 <= w_last - a.window)) {
#pragma unroll
      for (int n = 0; n < S::BN / 32; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int back = place - (k0 + 32 * n + 8 * (i >> 2) + 4 * half + (i & 3));
          if (back < 0 || (a.window > 0 && back >= a.window)) s[n][i] = -INFINITY;
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int n = 0; n < S::BN / 32; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[n][i]);
    st.follow(xor32_max(mx), a.c);
#pragma unroll
    for (int n = 0; n < S::BN / 32; ++n) st.add(st.weigh(s[n], a.c), V, 32 * n, lane);
  }
  const bool bad = PAGED && __syncthreads_or(x.bad);
  const float l = xor32_sum(st.l), f = bad ? NAN : (l == 0.f ? 0.f : 1.0f / l);
  if (row < rows) {
#pragma unroll
    for (int n = 0; n < C::NMB; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * n + 8 * g + 4 * half;
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = st.o[n][4 * g + i] * f;
        if (d < a.vchunks * C::E) *(typename Tile<T>::quad*)(out + d * (int)sizeof(T)) = to_quad<T>(v);
      }
  }
  if (!bad && __builtin_amdgcn_ballot_w64(st.odd())) {
    wait_vm<0>();  // what is above is written
    for (int r = w0; r < w0 + 32 && r < rows; ++r) {
      const int tk = r / a.group, hd = head * a.group + r - tk * a.group;
      seq_one<T, PAGED>(a, x, a.q + (sp.first + tk) * a.q_token + hd * a.q_head, a.out + (sp.first + tk) * a.o_token + hd * a.o_head,
                        place_of(r), lane);
    }
  }
}
}  // namespace khm
