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
// values, and l is the sum of the rounded ones: what is divided by it is a mean of the values, in which a weight's rounding weighs
// (v_j - out) and not v_j, so that a key that outweighs the others comes out as it is.  fp32 operands are split, not rounded (Split).
#pragma once
#include "kh_lgemm.h"

#include <type_traits>

namespace khm {
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

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
};

// fp32 on the bf16 matrix cores: a number is the sum of three of 8 bits, exactly - rounded to bf16, what is left rounded, what is left then.
// Of the nine products of two numbers the three smallest are left out, at most 2^-24 of the product each and of either sign: less than the
// fp32 matrix instruction's own rounding of n sums, for 6 x 32 cycles a block of 16 and not 8 x 64.  Numbers below 2^-110 have parts below the
// least there is, and keep fewer bits; those that bf16 has no room for end as no number, and their rows are done again.
struct Split {
  bf16x8 h, m, l;
};
__device__ __forceinline__ Split seq_split(const float (&x)[8]) {
  Split s;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    s.h[i] = (bf16)x[i];
    const float r = x[i] - (float)s.h[i];
    s.m[i] = (bf16)r;
    s.l[i] = (bf16)(r - (float)s.m[i]);
  }
  return s;
}
__device__ __forceinline__ Split seq_split(const f32x4& a, const f32x4& b) {
  const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  return seq_split(x);
}
// the products but the largest
__device__ __forceinline__ f32x16 mma_small(const Split& a, const Split& b, f32x16 c) {
  c = Tile32<bf16>::mma(a.l, b.h, c);
  c = Tile32<bf16>::mma(a.h, b.l, c);
  c = Tile32<bf16>::mma(a.m, b.m, c);
  c = Tile32<bf16>::mma(a.m, b.h, c);
  return Tile32<bf16>::mma(a.h, b.m, c);
}

// Where keys and values are.  Strides in bytes.
struct SeqKv {
  const char *k, *v;
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
  const int32_t* pages;  // nullptr: rows, those of the sequence's tokens
  int64_t table_stride;
  int n_pages, page_size, most;  // most: places of a sequence's row of the table
  uint32_t magic;  // place / page_size = umulhi(place, magic) >> shift; 0: page_size 1
  int shift;
  int plain;  // a request's rows are whole, in one page and evenly apart
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

// DP: elements of a row that are worked on, those behind a head's zeros in the queries and left out of the output.  A staged row has room
// for 64, 128 or 256; behind the head's own lies its last chunk again.  (What it holds meets zeros; where that gives what is no
// number, the row is done once more with care, as for any other.)
template <class T, int DP>
struct SeqCfg {
  static constexpr int E = 16 / (int)sizeof(T);
  static constexpr int RB = (DP <= 64 ? 64 : (DP <= 128 ? 128 : 256)) * (int)sizeof(T);  // bytes of a staged row
  static constexpr int CB = RB / 16;                    // its chunks
  static constexpr int NKB = DP * (int)sizeof(T) / 32;  // 32-byte k-blocks
  static constexpr int NMB = DP / 32;                   // 32-column blocks of the output
  static constexpr bool TIGHT = RB > 256 || sizeof(T) == 4;  // queries and outputs fill the registers: reads of LDS stay near their use
  static constexpr bool HOLD = RB <= 512;                    // queries in registers; else read, and split, again for each tile
  // LDS: chunk c of row r of the keys lies in slot c ^ turn_k(r), of the values in c ^ turn_v(r).  Reads of 16 bytes of 16 rows
  // (keys), of 32 bytes of four rows (values) then touch every bank once.  turn_v(r + 8) = turn_v(r), turn_v(4 + i) = turn_v(4) ^ turn_v(i),
  // turn_k(r + 16) = turn_k(r): a lane's addresses of a tile are one of its own, turned by constants.
  static __device__ __forceinline__ int turn_k(int r) { return RB == 128 ? (r >> 1) & 7 : r & 15; }
  static __device__ __forceinline__ int turn_v(int r) { return RB == 128 ? ((r >> 1) & 3) * 2 : (r & 7) * 2; }
};

template <class X>
__device__ __forceinline__ X lds_read(unsigned addr) {
  return *(const __attribute__((address_space(3))) X*)(size_t)addr;
}

// The same number, but nothing made of it is kept in registers over a loop
template <bool YES>
__device__ __forceinline__ int seq_fresh(int x) {
  if (YES) asm volatile("" : "+v"(x));
  return x;
}

// Numbers that are the same in every lane, where the compiler does not see it
__device__ __forceinline__ int seq_same(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t seq_same64(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)seq_same((int)(x >> 32)) << 32 | (uint32_t)seq_same((int)x));
}
__device__ __forceinline__ const char* seq_same(const char* p) { return (const char*)seq_same64((int64_t)p); }

// The running state of 32 query rows, a lane's row being l & 31.
template <class T, int DP>
struct SeqState {
  typedef SeqCfg<T, DP> C;
  typedef typename Tile32<T>::frag frag;
  // queries, by blocks of 32 bytes; fp32: by two of them
  static constexpr int PER = sizeof(T) == 2 ? 1 : 2;
  typename std::conditional<sizeof(T) == 2, frag, Split>::type q[C::HOLD ? C::NKB / PER : 1];
  const char* row;  // of the queries
  int chunks;
  f32x16 o[C::NMB];
  float m, l;  // l: this half's keys
  struct Rounded {  // the weights of 32 keys as their product with the values takes them
    bf16x8 p[2];
  };
  typedef typename std::conditional<sizeof(T) == 2, Rounded, f32x16>::type weights;
  // in the registers of the scores that they were
  static __device__ __forceinline__ f32x16 held(const weights& w) {
    if constexpr (sizeof(T) == 2) {
      f32x16 s = {};
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = __builtin_bit_cast(f32x4, w.p[i / 4])[i % 4];
      return s;
    } else {
      return w;
    }
  }
  static __device__ __forceinline__ weights taken(const f32x16& s) {
    if constexpr (sizeof(T) == 2) {
      weights w;
#pragma unroll
      for (int i = 0; i < 2; ++i) w.p[i] = __builtin_bit_cast(bf16x8, f32x4{s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]});
      return w;
    } else {
      return s;
    }
  }

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
    const int c = 2 * b + seq_fresh<C::TIGHT>(half);
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
      for (int b = 0; b < C::NKB / PER; ++b) {
        if constexpr (PER == 1) q[b] = query(b, half);
        else q[b] = seq_split(query(2 * b, half), query(2 * b + 1, half));
      }
  }
  // scores of 32 keys, rows r0 .. of the tile at K
  __device__ __forceinline__ f32x16 scores(unsigned K, int r0, int lane) const {
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
    const int r = lane & 31;
    const unsigned at = K + (unsigned)(r * C::RB + 16 * ((lane >> 5) ^ C::turn_k(r)));
    if constexpr (PER == 1) {
      constexpr int G = C::TIGHT ? 4 : C::NKB;  // requested together, the next ones ahead of these products
      frag k[2][G];
#pragma unroll
      for (int j = 0; j < G; ++j) k[0][j] = lds_read<frag>((at ^ (32 * j)) + r0 * C::RB);
#pragma unroll
      for (int g = 0; g < C::NKB / G; ++g) {
        if (g + 1 < C::NKB / G)
#pragma unroll
          for (int j = 0; j < G; ++j) k[(g + 1) & 1][j] = lds_read<frag>((at ^ (32 * (G * (g + 1) + j))) + r0 * C::RB);
#pragma unroll
        for (int j = 0; j < G; ++j) s = Tile32<T>::mma(k[g & 1][j], q[G * g + j], s);
        if (C::TIGHT) __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      f32x16 small = s;  // apart: as many roundings of the sum as it has blocks
#pragma unroll
      for (int b = 0; b < C::NKB / 2; ++b) {
        const Split k = seq_split(lds_read<frag>((at ^ (64 * b)) + r0 * C::RB), lds_read<frag>((at ^ (64 * b + 32)) + r0 * C::RB));
        const Split& x = C::HOLD ? q[C::HOLD ? b : 0] : seq_split(query(2 * b, lane >> 5), query(2 * b + 1, lane >> 5));
        small = mma_small(k, x, small);
        s = Tile32<bf16>::mma(k.h, x.h, s);
        if (b % 2 == 1) __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] += small[i];
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
  __device__ __forceinline__ weights weigh(const f32x16& s, float c) {
    const float base = m == -INFINITY ? 0.f : -m * c;  // no key seen yet: 2^-inf
    f32x16 p;
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, base));
    float t = 0.f;
    if constexpr (sizeof(T) == 2) {
      weights w;
#pragma unroll
      for (int i = 0; i < 16; ++i) w.p[i / 8][i % 8] = (bf16)p[i];
      // two of them a sum, off by 2^-23 of it at most
      const bf16x2 ones = {(bf16)1.f, (bf16)1.f};
#pragma unroll
      for (int i = 0; i < 16; i += 2) t = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{w.p[i / 8][i % 8], w.p[i / 8][i % 8 + 1]}, ones, t, false);
      l += t;
      return w;
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) t += p[i];
      l += t;
      return p;
    }
  }
  // O^T += V^T P^T for 32 keys, rows r0 .. of the tile at V
  __device__ __forceinline__ void add(const weights& w, unsigned V, int r0, int lane) {
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      const int r = 4 * half + ((lane >> 2) & 3);  // of eight
      const unsigned at = V + (unsigned)(r * C::RB + 16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ C::turn_v(r)) + 8 * (lane & 1));
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        constexpr int G = C::TIGHT ? 2 : C::NMB;
        bf16x8 a[2][G];
        auto load = [&](int g) __attribute__((always_inline)) {
#pragma unroll
          for (int j = 0; j < G; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const bf16x4 v = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(size_t)((at ^ (64 * (G * g + j))) + (r0 + 16 * t + 8 * e) * C::RB)));
#pragma unroll
              for (int i = 0; i < 4; ++i) a[g & 1][j][4 * e + i] = v[i];
            }
        };
        load(0);
#pragma unroll
        for (int g = 0; g < C::NMB / G; ++g) {
          if (g + 1 < C::NMB / G) load(g + 1);
#pragma unroll
          for (int j = 0; j < G; ++j) o[G * g + j] = Tile32<T>::mma(a[g & 1][j], w.p[t], o[G * g + j]);
          if (C::TIGHT) __builtin_amdgcn_sched_barrier(0);
        }
      }
    } else {
      const unsigned at = V + (unsigned)(4 * half * C::RB + 16 * (((lane & 31) >> 2) ^ C::turn_v(4 * half)) + 4 * (lane & 3));
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = w[8 * t + j];
        const Split x = seq_split(p);
#pragma unroll
        for (int n = 0; n < C::NMB; ++n) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            v[j] = lds_read<float>((at ^ (16 * C::turn_v(j & 3) + 128 * n)) + (r0 + 16 * t + 8 * (j >> 2) + (j & 3)) * C::RB);
          const Split y = seq_split(v);
          o[n] = Tile32<bf16>::mma(y.h, x.h, mma_small(y, x, o[n]));
          __builtin_amdgcn_sched_barrier(0);
        }
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

__device__ __forceinline__ int seq_chunk(int c, int chunks) { return c < chunks ? c : chunks - 1; }

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
__device__ __forceinline__ int seq_page(const SeqKv& kv, int place) {
  return kv.magic ? (int)(__umulhi((uint32_t)place, kv.magic) >> kv.shift) : place;
}
// A sequence's pages are looked up SEQ_TAB at a time, into LDS: an address then waits for no memory, and above all not for the
// requests under way, which a load of its own would have to let pass.
constexpr int SEQ_TAB = 1024;
constexpr int SEQ_SHARES = 512;  // the most that work is dealt to: two workgroups on each of MI355X's 256 CUs
// Steps of `keys` keys that surely need no more pages than the table holds.
__device__ __forceinline__ int seq_table_steps(const SeqKv& kv, int keys) {
  const int64_t n = (int64_t)(SEQ_TAB - 1) * kv.page_size / keys;
  return n < 1 << 20 ? (int)n : 1 << 20;
}
// The pages of keys [ka, kb); *bad where one is outside the cache.  Barriers before and after are the caller's.
__device__ __forceinline__ int seq_table(const SeqKv& kv, const int32_t* table, int ka, int kb, int* tab, int* bad) {
  const int p0 = seq_page(kv, ka), n = seq_page(kv, kb - 1) - p0 + 1;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int page = table[p0 + i];
    const bool ok = (unsigned)page < (unsigned)kv.n_pages;
    tab[i] = ok ? page : 0;
    if (!ok) *bad = 1;
  }
  return p0;
}

// One query by one wave from global memory, 64 keys at a time, in two passes: the maximum and the sum of the weights, then the values,
// each with its weight over that sum, which is at most 1 - so that no sum of them passes what a number holds where their mean does not.
// A lane has a key for the scores, four columns for the output.  A key that the query does not see is not touched, so that what
// it holds cannot reach it (in a product over a tile it is zero times the value, which is no zero for what is no number): for the
// rows where that seems to have happened, and for those whose weights add up to nothing though they see a key (its place is theirs):
// c times their scores has no room in a number, or all of these are minus infinity, and the row is NaN, as of the formula.
template <class T, bool PAGED>
__device__ __forceinline__ void seq_one(const SeqArgs& a, SeqKeys& x, const char* q, char* out, int place, int lane_) {
  typedef typename Tile<T>::frag frag;
  constexpr int E = Tile<T>::N, DEEP = 8;  // keys whose values are requested together
  const int lane = seq_fresh<true>(lane_);  // nothing of this in registers over the caller's loop
  const int lo = a.window > 0 && place >= a.window ? place - a.window + 1 : 0, cols = a.vchunks * E;
  auto score = [&](int key, int64_t& vo) __attribute__((always_inline)) {
    float s = -INFINITY;
    if (key <= place) {
      int64_t ko;
      seq_row<PAGED>(a, x, key, ko, vo);
      s = 0.f;
#pragma unroll 4
      for (int c = 0; c < a.kchunks; ++c) {
        const frag u = *(const frag*)(q + 16 * c), w = *(const frag*)(x.k + ko + 16 * c);
        for (int i = 0; i < E; ++i) s = __builtin_fmaf((float)u[i], (float)w[i], s);
      }
    }
    return s;
  };
  float m = -INFINITY, l = 0.f;  // l: this lane's keys
  // the scores' difference first: c times a score may have no room
  auto weight = [&](float s) __attribute__((always_inline)) { return s == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((s - m) * a.c); };
  int64_t vo = 0;
  for (int k0 = lo; k0 <= place; k0 += 64) {
    const float s = score(k0 + lane, vo), before = m;
    m = fmaxf(m, wave_max(s));
    l = l * (before == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((before - m) * a.c)) + weight(s);
  }
  l = wave_sum(l);
  const bool bad = __builtin_amdgcn_ballot_w64(x.bad) != 0;
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  if (bad || l != l || (l == 0.f && place >= 0)) {
    for (int i = 0; i < 4; ++i) o[i] = NAN;
  } else if (l != 0.f) {
    const float share = 1.0f / l;
    for (int k0 = lo; k0 <= place; k0 += 64) {
      const float p = weight(score(k0 + lane, vo)) * share;
      const int n = place - k0 < 63 ? place - k0 + 1 : 64;
      for (int j0 = 0; j0 < n; j0 += DEEP) {
        T v[DEEP][4];  // the last key and column again where there are no more: a load that nothing has to decide about waits for nothing
#pragma unroll
        for (int j = 0; j < DEEP; ++j) {
          const T* row = (const T*)(x.v + __shfl((long long)vo, j0 + j < n ? j0 + j : n - 1));
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (64 * i < cols) v[j][i] = row[lane + 64 * i < cols ? lane + 64 * i : cols - 1];
        }
#pragma unroll
        for (int j = 0; j < DEEP; ++j) {
          if (j0 + j >= n) continue;
          const float w = __shfl(p, j0 + j);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (64 * i < cols) o[i] = __builtin_fmaf(w, (float)v[j][i], o[i]);
        }
      }
    }
  }
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < cols) ((T*)out)[lane + 64 * i] = (T)o[i];
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
  static constexpr int RING = 4 * TB;                // two tiles of keys and values each
  static constexpr int MOST = 1024;                  // slots that are looked at to be cut
  static constexpr int LDS_PACKED = RING, LDS_PAGED = RING + 4 * SEQ_TAB + 64, LDS_SHARES = LDS_PAGED + 4 * (MOST + 4);
  static constexpr int LEAST = 512 / BN;             // steps of a part: 64 tokens behind 4032 keys 33 us, by 256 keys 38, by 1024 37
};

// 128 query rows of a key head, as one of four waves sees them.
struct SeqTile {
  SeqSpan sp;
  SeqKeys x;
  int b, head, rows, w0, row, token, h, place, w_first, w_last, t_lo, t_hi;  // tiles of keys [t_lo, t_hi)
};
template <int BM, int BN, bool PAGED>
__device__ __forceinline__ bool seq_tile(const SeqArgs& a, int slot, int head, SeqTile& s, int wave, int lane) {
  s.b = __builtin_amdgcn_readfirstlane(seq_of_slot(a, slot, BM, lane));
  s.head = head;
  s.sp = seq_span(a, s.b);
  s.rows = s.sp.n * a.group;
  if (PAGED && s.rows <= 32) return false;  // k_seq_rows
  // long tiles of a sequence first
  const int tiles = (s.rows + BM - 1) / BM, tile = tiles - 1 - (slot - seq_slot_base(a, s.b, BM));
  if (tile < 0 || tile >= tiles) return false;
  auto place_of = [&](int r) __attribute__((always_inline)) { return s.sp.length - s.sp.n + (r < s.rows ? r : s.rows - 1) / a.group; };
  const int r0 = tile * BM;
  s.w0 = r0 + 32 * wave;
  s.row = s.w0 + (lane & 31);
  s.x = seq_keys(a, s.b, head, s.sp, place_of(r0), place_of(r0 + BM - 1));
  s.w_first = place_of(s.w0);
  s.w_last = place_of(s.w0 + 31);
  s.place = place_of(s.row);
  const int r = s.row < s.rows ? s.row : s.rows - 1;
  s.token = r / a.group;
  s.h = head * a.group + r - s.token * a.group;
  s.t_lo = s.x.lo / BN;
  s.t_hi = (s.x.hi + BN - 1) / BN;
  return true;
}
// Tiles [t0, t1) of keys, shared by the four waves, into the state.  tab, bad: of pages (LDS).
template <class T, int DP, bool PAGED>
__device__ __forceinline__ void seq_tile_run(const SeqArgs& a, const SeqTile& s, SeqState<T, DP>& st, int t0, int t1, unsigned lds0, int* tab, int* bad,
                                             int wave, int lane) {
  typedef SeqTiles<T, DP> S;
  typedef SeqCfg<T, DP> C;
  constexpr int NL = S::BN * C::CB / (64 * S::W);
  static_assert(NL * 64 * S::W == S::BN * C::CB, "whole requests");
  t0 = __builtin_amdgcn_readfirstlane(t0);
  t1 = __builtin_amdgcn_readfirstlane(t1);
  const char *kp = seq_same(s.x.k), *vp = seq_same(s.x.v);
  const int half = lane >> 5, most = PAGED ? seq_table_steps(a.kv, S::BN) : t1 - t0;
  for (int c0 = t0; c0 < t1; c0 += most) {
    const int c1 = t1 - c0 < most ? t1 : c0 + most;
    const int ka = seq_same(c0 * S::BN > s.x.lo ? c0 * S::BN : s.x.lo), kb = seq_same(c1 * S::BN < s.x.hi ? c1 * S::BN : s.x.hi);
    int p0 = 0;
    if constexpr (PAGED) {
      __syncthreads();
      p0 = seq_same(seq_table(a.kv, s.x.table, ka, kb, tab, bad));
      __syncthreads();
    }
    auto issue = [&](int t) __attribute__((always_inline)) {
      const unsigned K = lds0 + (unsigned)((t & 1) * 2 * S::TB), V = K + S::TB;
      if (a.kv.plain && t * S::BN >= ka && t * S::BN + S::BN <= kb) {  // addresses in the scalar unit: one lane's offset serves every request
        constexpr int RPR = 64 / C::CB;  // rows of a request
        const int r = lane / C::CB, c = lane % C::CB;
#pragma unroll
        for (int j = 0; j < NL; ++j) {
          const int row = (S::W * j + wave) * RPR, place = t * S::BN + row;
          const char *k = kp, *v = vp;
          if constexpr (PAGED) {
            const int p = seq_page(a.kv, place), page = seq_same(tab[p - p0]), slot = place - p * a.kv.page_size;
            k += page * a.kv.k_page + slot * a.kv.k_slot;
            v += page * a.kv.v_page + slot * a.kv.v_slot;
          } else {
            k += place * a.kv.k_slot;
            v += place * a.kv.v_slot;
          }
          const unsigned at = (unsigned)((S::W * j + wave) * 1024);
          dma_x4_keep(k, (unsigned)(r * (int)a.kv.k_slot + 16 * seq_chunk(c ^ C::turn_k(row + r), a.kchunks)), K + at);
          dma_x4_keep(v, (unsigned)(r * (int)a.kv.v_slot + 16 * seq_chunk(c ^ C::turn_v(row + r), a.vchunks)), V + at);
        }
        return;
      }
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int i = (S::W * j + wave) * 64 + seq_fresh<C::TIGHT>(lane), r = i / C::CB, c = i - r * C::CB, ck = c ^ C::turn_k(r), cv = c ^ C::turn_v(r);
        int place = t * S::BN + r;
        place = place < ka ? ka : (place >= kb ? kb - 1 : place);
        int64_t ko, vo;
        if constexpr (PAGED) {
          const int p = seq_page(a.kv, place), slot = place - p * a.kv.page_size, page = tab[p - p0];
          ko = page * a.kv.k_page + slot * a.kv.k_slot;
          vo = page * a.kv.v_page + slot * a.kv.v_slot;
        } else {
          ko = place * a.kv.k_slot;
          vo = place * a.kv.v_slot;
        }
        const unsigned at = (unsigned)((S::W * j + wave) * 1024);
        dma_x4_from(s.x.k + ko + 16 * seq_chunk(ck, a.kchunks), K + at);
        dma_x4_from(s.x.v + vo + 16 * seq_chunk(cv, a.vchunks), V + at);
        if (C::TIGHT) __builtin_amdgcn_sched_barrier(0);
      }
    };
    issue(c0);
    for (int t = c0; t < c1; ++t) {
      wait_vm<0>();     // this tile has landed
      __syncthreads();  // for every wave, and everyone is done with the tile before
      if (t + 1 < c1) issue(t + 1);
      const int k0 = t * S::BN;
      if (k0 > s.w_last || (a.window > 0 && k0 + S::BN - 1 <= s.w_first - a.window)) continue;  // nothing that this wave sees
      const unsigned K = lds0 + (unsigned)((t & 1) * 2 * S::TB), V = K + S::TB;
      f32x16 p[S::BN / 32];
#pragma unroll
      for (int n = 0; n < S::BN / 32; ++n) p[n] = st.scores(K, 32 * n, lane);
      if (k0 + S::BN - 1 > s.w_first || (a.window > 0 && k0 <= s.w_last - a.window)) {
#pragma unroll
        for (int n = 0; n < S::BN / 32; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int back = s.place - (k0 + 32 * n + 8 * (i >> 2) + 4 * half + (i & 3));
            if (back < 0 || (a.window > 0 && back >= a.window)) p[n][i] = -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < S::BN / 32; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, p[n][i]);
      st.follow(xor32_max(mx), a.c);
#pragma unroll
      for (int n = 0; n < S::BN / 32; ++n) st.add(st.weigh(p[n], a.c), V, 32 * n, lane);
    }
  }
}
// The wave's 32 rows, l being those of both halves; rows with what is no number, and they alone, once more, with care.
template <class T, int DP, bool PAGED>
__device__ __forceinline__ void seq_tile_write(const SeqArgs& a, SeqTile& s, const SeqState<T, DP>& st, float l, bool bad, int lane) {
  typedef SeqCfg<T, DP> C;
  const float f = bad ? NAN : (l == 0.f ? 0.f : 1.0f / l);
  if (s.row < s.rows) {
    char* out = a.out + (s.sp.first + s.token) * a.o_token + s.h * a.o_head;
#pragma unroll
    for (int n = 0; n < C::NMB; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * n + 8 * g + 4 * (lane >> 5);
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = st.o[n][4 * g + i] * f;
        if (d < a.vchunks * C::E) *(typename Tile<T>::quad*)(out + d * (int)sizeof(T)) = to_quad<T>(v);
      }
  }
  const uint64_t odd = __builtin_amdgcn_ballot_w64(!bad && s.row < s.rows && (st.odd() || (l == 0.f && s.place >= 0)));
  if (odd) {
    wait_vm<0>();  // what is above is written
    s.x.bad = false;
    for (uint32_t left = (uint32_t)(odd | odd >> 32); left; left &= left - 1) {
      const int r = s.w0 + __builtin_ctz(left), tk = r / a.group, hd = s.head * a.group + r - tk * a.group;
      seq_one<T, PAGED>(a, s.x, a.q + (s.sp.first + tk) * a.q_token + hd * a.q_head, a.out + (s.sp.first + tk) * a.o_token + hd * a.o_head,
                        s.sp.length - s.sp.n + tk, lane);
    }
  }
}

// Four waves of 32 rows each share the tiles of keys and values.  grid (slots * kv_heads): the key heads side by side, so that a
// key head's tiles stay with one XCD's L2 where their number is a multiple of eight.  8192 tokens of 32 heads over 8: 308 us at heads of
// 64 (893 TFLOP/s; the chip clocks down to 1.82 GHz, the matrix cores are busy 43 % of its cycles, the vector unit with its exponentials and
// maxima 67), 575 at 128 (956; 2.0 GHz, 45 and 40).
template <class T, int DP, bool PAGED>
__global__ __launch_bounds__(256, DP <= 64 && sizeof(T) == 2 ? 3 : (DP <= 128 ? 2 : 1)) void k_seq_tiles(const SeqArgs a) {
  typedef SeqTiles<T, DP> S;
  extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
  int *tab = (int*)(smem_raw + S::RING), *bad = tab + SEQ_TAB;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = (int)blockIdx.x % a.kv_heads, slot = (int)blockIdx.x / a.kv_heads;
  SeqTile s;
  if (!seq_tile<S::BM, S::BN, PAGED>(a, slot, head, s, wave, lane)) return;
  if (PAGED && threadIdx.x == 0) *bad = s.x.bad;
  SeqState<T, DP> st;
  st.load_q(a.q + (s.sp.first + s.token) * a.q_token + s.h * a.q_head, lane >> 5, a.kchunks);
  st.clear();
  seq_tile_run<T, DP, PAGED>(a, s, st, s.t_lo, s.t_hi, (unsigned)__builtin_amdgcn_readfirstlane((int)kh_lds_addr(smem_raw)), tab, bad, wave, lane);
  if (PAGED) __syncthreads();
  seq_tile_write<T, DP, PAGED>(a, s, st, xor32_sum(st.l), PAGED && *bad, lane);
}

// ---- few rows a sequence ---------------------------------------------------------------------------------------------------------
// Sequences of up to 32 query rows (single tokens above all) read their keys once, whatever is done: memory bounds them, so all keys
// of all sequences are dealt evenly to the workgroups that fit on the chip at once.  One token over 131072 keys of 8 heads of 64
// 61.5 us, 64 over 90 - 8106 keys of 8 heads of 128 115: 4.4 TB/s, not far from a copy's rate; requests alone, by the same instruction, have reached
// 5.9 and, as read once, 7.1, and what lies between is not told apart.  A unit is a key head of a sequence; units lie one
// behind the other, each a head and a number of steps of 128 keys, and workgroup i takes places [i W / N, (i + 1) W / N) of the W, the
// end of one unit and the beginning of the next where they fall so.  What it finds of a unit that others have parts of goes to
// the workspace, fp32 and with its m and l; the workgroup that is the last to bring a part adds them, in the order of the keys whoever
// it is.  Every workgroup finds its share from the lengths on the device by one sum over the sequences: no table from the host, and a
// captured launch follows the lengths.
struct SeqRowsArgs {
  SeqArgs s;
  // [N] parts brought of the unit that begins in workgroup i's share and ends behind it, 0 between launches
  int* brought;
  float* ws;        // [2 N][32][value size + 4], o, m, l: of the unit that began before workgroup i's share, of the one that ends behind it
  int all;          // sequences of more than 32 rows too, 32 at a time
  // the same for tiles of many rows
  int* brought_tiles;
  float* ws_tiles;
};
struct SeqUnits {
  SeqSpan sp;
  int rows, blocks, lo, hi, t0, steps;  // of each of blocks * kv_heads units
  int64_t all;                          // places of all of them
};
constexpr int SEQ_STEP = 128;     // four waves of 32 keys
// Places ahead of a unit's first step, for what a unit costs beside its steps: 256 tokens over 100 - 1885 keys at heads of 64, the short ones
// first, take 169 us without, 109 with 1, 111 with 2, 121 with 5.
constexpr int SEQ_HEAD = 1;
__device__ __forceinline__ SeqUnits seq_units(const SeqRowsArgs& a, int b) {
  SeqUnits u;
  u.sp = seq_span(a.s, b);
  u.rows = u.sp.n * a.s.group;
  u.blocks = u.rows <= 32 || a.all ? (u.rows + 31) / 32 : 0;
  const int first = u.sp.length - u.sp.n;
  u.lo = a.s.window > 0 && first >= a.s.window ? first - a.s.window + 1 : 0;
  u.hi = u.sp.length;
  u.t0 = u.lo / SEQ_STEP;
  const int n = (u.hi + SEQ_STEP - 1) / SEQ_STEP - u.t0;
  u.steps = n > 1 ? n : 1;  // no key at all: a step that writes the zeros
  u.all = (int64_t)u.blocks * a.s.kv_heads * (u.steps + SEQ_HEAD);
  return u;
}
// Steps ahead of each sequence and in all, for a workgroup of 256.  A thread sums `per` sequences that lie side by side.
struct SeqScan {
  int64_t before, mine, total;  // of this thread's sequences
  int per;
};
__device__ __forceinline__ SeqScan seq_scan(const SeqRowsArgs& a, int64_t* red /* [4] */) {
  SeqScan r;
  r.per = (a.s.n_seqs + 255) / 256;
  r.mine = 0;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b0 = (int)threadIdx.x * r.per;
  for (int b = b0; b < b0 + r.per && b < a.s.n_seqs; ++b) {
    const SeqUnits u = seq_units(a, b);
    r.mine += u.all;
  }
  int64_t x = r.mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t y = __shfl_up((long long)x, d);
    if (lane >= d) x += y;
  }
  if (lane == 63) red[wave] = x;
  __syncthreads();
  r.before = x - r.mine;
  r.total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) r.before += red[w];
    r.total += red[w];
  }
  return r;
}
// Of N workgroups, those that have work, and where the share of one begins.
__device__ __forceinline__ int seq_shares(int64_t total, int n) { return total < n ? (int)total : n; }
__device__ __forceinline__ int64_t seq_share(int64_t total, int n, int i) { return total * i / n; }
// The workgroup that has the first part of a unit of rows, and the number of its parts, those of the workgroups that follow: one more than the
// borders behind its head.
__device__ __forceinline__ int seq_parts(int64_t total, int n, int64_t unit, int places, int& first) {
  const int64_t y = unit + SEQ_HEAD + 1, z = unit + places - 1;
  const int a = (int)((y * n + total - 1) / total), b = (int)(((z + 1) * n + total - 1) / total) - 1;
  first = a - 1;
  return b < a ? 1 : b - a + 2;
}

template <class T, int DP>
struct SeqRows {
  typedef SeqCfg<T, DP> C;
  static constexpr int TB = 32 * C::RB;  // keys of a wave's tile, or their values
  // A wave has a ring of such halves of its own: keys, values, keys ..., as many as leave the CU its other waves
  static constexpr int NB = C::RB <= 128 ? 4 : (C::RB <= 512 ? 2 : 1);
  static constexpr int NL = 32 * C::CB / 64;  // requests for one
  static constexpr int PITCH = DP + 1;        // of a row of partial outputs, in the same place
  static constexpr int RING = 4 * NB * TB > 16 * 32 * PITCH ? 4 * NB * TB : 16 * 32 * PITCH;
  static constexpr int LDS = RING + 4 * SEQ_TAB + 1024 + 64;
  static_assert(4 * SEQ_SHARES <= RING && 4096 <= 4 * SEQ_TAB, "a row's weights fit the ring, the sums of parts the table");
  static constexpr int SHARES = LDS <= 80 * 1024 ? SEQ_SHARES : SEQ_SHARES / 2;
};

// Rows of a unit, a bit each, once more with care, by the waves in turn.
template <class T, bool PAGED>
__device__ __forceinline__ void seq_finish(const SeqArgs& a, const SeqUnits& u, int b, int head, int r0, uint32_t odd, int wave, int lane) {
  for (int i = 0; odd; ++i, odd &= odd - 1) {
    if (i % 4 != wave) continue;
    const int r = r0 + __builtin_ctz(odd), tk = r / a.group, h = head * a.group + r - tk * a.group, place = u.sp.length - u.sp.n + tk;
    SeqKeys x = seq_keys(a, b, head, u.sp, place, place);
    seq_one<T, PAGED>(a, x, a.q + (u.sp.first + tk) * a.q_token + h * a.q_head, a.out + (u.sp.first + tk) * a.o_token + h * a.o_head, place, lane);
  }
}

// Partial results pass between workgroups, maybe of different XCDs, in words of agent scope, which are stored through and read past the
// caches that are not common (a fence for each part instead costs a launch of 512 workgroups 15 - 20 us), four at a time: an atomic load
// has one, and the joining workgroup waits for as many requests as it can have under way.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ __amdgpu_buffer_rsrc_t seq_parts_at(float* p) { return __builtin_amdgcn_make_buffer_rsrc(p, 0, 0x7fffffff, 0x00020000); }
constexpr int SEQ_AGENT = 16;  // sc1
__device__ __forceinline__ void seq_give(__amdgpu_buffer_rsrc_t to, unsigned at, const f32x4& v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), to, (int)(4 * at), 0, SEQ_AGENT);
}
__device__ __forceinline__ f32x4 seq_take(__amdgpu_buffer_rsrc_t from, unsigned at) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, (int)(4 * at), 0, SEQ_AGENT));
}

// The rows of a unit from its parts: their weights (LDS, as many rows at a time as fit `room` floats), then their outputs, four columns a
// thread and as many parts side by side as there are threads.  -> this thread's rows, a bit each, whose output is no number
template <class T>
__device__ __forceinline__ uint32_t seq_join(const SeqRowsArgs& ra, const SeqUnits& u, int head, int r0, int n_rows, int i0, int parts, float* weight,
                                         int room, float* ls, f32x4* red, int wave, int lane) {
  const SeqArgs& a = ra.s;
  const int cols = a.vchunks * (16 / (int)sizeof(T)), pitch = cols + 4;
  // part p: the end of workgroup i0's share for the first, the beginning of that of i0 + p for the others
  auto at = [&](int r, int p) __attribute__((always_inline)) { return (unsigned)(((2 * (i0 + p) + (p == 0 ? 1 : 0)) * 32 + r) * pitch); };
  const __amdgpu_buffer_rsrc_t ws = seq_parts_at(ra.ws);
  int across = 1, down = 1;  // threads of a row: its columns by four; rows at once
  while (across * 4 < cols) across *= 2;
  while (down < n_rows && down * across < 256 && 2 * down * parts <= room) down *= 2;
  const int side = 256 / (across * down), x = (int)threadIdx.x & (across - 1), y = (int)threadIdx.x / across & (down - 1),
            z = (int)threadIdx.x / (across * down);
  uint32_t odd = 0;
  for (int rb = 0; rb < n_rows; rb += down) {
    for (int r = rb + wave; r < rb + down && r < n_rows; r += 4) {
      constexpr int PER = SEQ_SHARES / 64;
      float mp[PER], lp[PER], m = -INFINITY, l = 0.f;  // all requested together
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        mp[k] = -INFINITY;
        lp[k] = 0.f;
        if (lane + 64 * k < parts) {
          const f32x4 ml = seq_take(ws, at(r, lane + 64 * k) + cols);
          mp[k] = ml[0];
          lp[k] = ml[1];
        }
      }
#pragma unroll
      for (int k = 0; k < PER; ++k) m = fmaxf(m, mp[k]);
      m = wave_max(m);
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const float f = mp[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mp[k] - m) * a.c);
        if (lane + 64 * k < parts) weight[(r - rb) * parts + lane + 64 * k] = f;
        l += mp[k] == -INFINITY ? lp[k] : lp[k] * f;  // NaN of a page that is none
      }
      l = wave_sum(l);
      if (lane == 0) ls[r] = l;
    }
    __syncthreads();
    const int r = rb + y;
    const bool mine = r < n_rows && 4 * x < cols;
    f32x4 o = f4_zero();
    if (mine) {
      constexpr int DEEP = 8;  // parts requested together
      for (int p = z; p < parts; p += DEEP * side) {
        f32x4 v[DEEP];
#pragma unroll
        for (int k = 0; k < DEEP; ++k) v[k] = p + k * side < parts ? seq_take(ws, at(r, p + k * side) + 4 * x) : f4_zero();
#pragma unroll
        for (int k = 0; k < DEEP; ++k) {
          const float f = p + k * side < parts ? weight[y * parts + p + k * side] : 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(v[k][i], f, o[i]);
        }
      }
    }
    red[threadIdx.x] = o;
    __syncthreads();
    if (mine && z == 0) {
      for (int p = 1; p < side && p < parts; ++p) {
        const f32x4 v = red[p * across * down + threadIdx.x];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += v[i];
      }
      const float l = ls[r];
      const int tk = (r0 + r) / a.group, hd = head * a.group + r0 + r - tk * a.group;
      bool again = l == 0.f && u.sp.length - u.sp.n + tk >= 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i] = l == 0.f ? 0.f : o[i] / l;
        again |= !(fabsf(o[i]) < INFINITY);
      }
      odd |= (uint32_t)again << r;
      *(typename Tile<T>::quad*)(a.out + (u.sp.first + tk) * a.o_token + hd * a.o_head + 4 * x * (int)sizeof(T)) = to_quad<T>(o);
    }
    __syncthreads();
  }
  return odd;
}

// Workgroup `share` of `shares`; whole prompts: 32 rows of a key head, slot of 32 rows by slot
template <class T, int DP, bool PAGED>
__device__ __forceinline__ void seq_rows(const SeqRowsArgs& ra, int shares, int share, char* smem_raw) {
  typedef SeqRows<T, DP> S;
  typedef SeqCfg<T, DP> C;
  int* tab = (int*)(smem_raw + S::RING);
  float *ms = (float*)(tab + SEQ_TAB), *ls = ms + 128;
  int64_t* red = (int64_t*)(ls + 128);
  int* flag = (int*)(red + 4);
  const SeqArgs& a = ra.s;
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned lds0 = (unsigned)__builtin_amdgcn_readfirstlane((int)kh_lds_addr(smem_raw));
  const unsigned ring = lds0 + (unsigned)(wave * S::NB * S::TB);
  // ---- this workgroup's share
  SeqScan sc;
  SeqUnits u;
  int n_shares = 1, b = 0, head = 0, r0 = 0, ta = 0, tb = 0, places = 0, unit = 0;
  int64_t at = 0, end = 1, ahead = 0;  // ahead: places ahead of sequence b
  if constexpr (PAGED) {
    sc = seq_scan(ra, red);
    n_shares = seq_shares(sc.total, shares);
    if (share >= n_shares) return;
    at = seq_share(sc.total, n_shares, share);
    end = seq_share(sc.total, n_shares, share + 1);
    if (sc.before <= at && at < sc.before + sc.mine) {  // one thread
      int64_t p = sc.before;
      int b = (int)threadIdx.x * sc.per;
      for (;; ++b) {
        const int64_t n = seq_units(ra, b).all;
        if (at < p + n) break;
        p += n;
      }
      flag[0] = b;
      *(int64_t*)(flag + 2) = p;
    }
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(flag[0]);
    ahead = *(int64_t*)(flag + 2);
    u = seq_units(ra, b);
  } else {
    const int slot = share / a.kv_heads;
    b = seq_same(seq_of_slot(a, slot, 32, lane));
    u.sp = seq_span(a, b);
    u.rows = u.sp.n * a.group;
    u.blocks = (u.rows + 31) / 32;
    head = share - slot * a.kv_heads;
    r0 = 32 * (u.blocks - 1 - (slot - seq_slot_base(a, b, 32)));  // long ones first
    if (r0 < 0 || r0 >= u.rows) return;
    const int first = r0 / a.group, last = (r0 + 31 < u.rows ? r0 + 31 : u.rows - 1) / a.group;
    u.lo = a.window > 0 && first >= a.window ? first - a.window + 1 : 0;
    u.hi = last + 1;
    u.t0 = u.lo / SEQ_STEP;
    tb = u.steps = (u.hi + SEQ_STEP - 1) / SEQ_STEP - u.t0;
  }
  int p0 = 0, tab_b = -1, tab_ka = 0, tab_kb = 0;  // the table holds the pages of keys [tab_ka, tab_kb) of tab_b, from page p0 on
  while (at < end) {
    if constexpr (PAGED) {
      while (at >= ahead + u.all) {
        ahead += u.all;
        u = seq_units(ra, ++b);
      }
      places = u.steps + SEQ_HEAD;
      unit = (int)((at - ahead) / places);
      const int from = (int)((at - ahead) - (int64_t)unit * places), to = places - from < end - at ? places : from + (int)(end - at);
      at += to - from;
      ta = from > SEQ_HEAD ? from - SEQ_HEAD : 0;
      tb = to > SEQ_HEAD ? to - SEQ_HEAD : 0;
      if (tb <= ta) continue;  // nothing but the unit's head: the workgroup that follows begins it
      head = unit / u.blocks;
      r0 = 32 * (unit - head * u.blocks);
    } else {
      at = end;
    }
    const int n_rows = u.rows - r0 < 32 ? u.rows - r0 : 32;
    const int row = r0 + ((lane & 31) < n_rows ? (lane & 31) : n_rows - 1);
    const int token = row / a.group, h = head * a.group + row - token * a.group, place = u.sp.length - u.sp.n + token;
    const int first_place = u.sp.length - u.sp.n + r0 / a.group, last_place = u.sp.length - u.sp.n + (r0 + n_rows - 1) / a.group;
    SeqKeys x = seq_keys(a, b, head, u.sp, u.sp.length - u.sp.n, u.sp.length - 1);
    const char *kp = seq_same(x.k), *vp = seq_same(x.v);
    SeqState<T, DP> st;
    st.load_q(a.q + (u.sp.first + token) * a.q_token + h * a.q_head, half, a.kchunks);
    st.clear();
    if (PAGED && threadIdx.x == 0 && b != tab_b) flag[1] = x.bad;  // and stays set for the sequence: nothing of it is a number then
    const int per_table = PAGED ? seq_table_steps(a.kv, SEQ_STEP) : tb - ta;
    for (int c0 = ta; c0 < tb && u.hi > u.lo; c0 += per_table) {
      const int c1 = tb - c0 < per_table ? tb : c0 + per_table;
      const int ka = (u.t0 + c0) * SEQ_STEP > u.lo ? (u.t0 + c0) * SEQ_STEP : u.lo, kb = (u.t0 + c1) * SEQ_STEP < u.hi ? (u.t0 + c1) * SEQ_STEP : u.hi;
      __syncthreads();  // the table before, and partial outputs, are read
      if (PAGED && (b != tab_b || ka != tab_ka || kb > tab_kb)) {  // not that of the key head before
        p0 = seq_table(a.kv, x.table, ka, kb, tab, flag + 1);
        tab_b = b;
        tab_ka = ka;
        tab_kb = kb;
        __syncthreads();
      }
      // half h of these steps: the keys (h even) or the values of step h / 2
      const int halves = 2 * (c1 - c0);
      auto issue = [&](int h) __attribute__((always_inline)) {
        const int k0 = seq_same((u.t0 + c0 + (h >> 1)) * SEQ_STEP + 32 * wave);
        const unsigned dst = ring + (unsigned)(h % S::NB * S::TB);
        const bool keys = (h & 1) == 0;
        const char* base = keys ? kp : vp;
        const int64_t ps = keys ? a.kv.k_page : a.kv.v_page, ss = keys ? a.kv.k_slot : a.kv.v_slot;
        const int chunks = keys ? a.kchunks : a.vchunks;
        if (a.kv.plain && k0 >= ka && k0 + 32 <= kb) {  // addresses in the scalar unit
          constexpr int RPR = 64 / C::CB;
          const int r = seq_fresh<C::TIGHT>(lane) / C::CB, c = lane % C::CB;
#pragma unroll
          for (int j = 0; j < S::NL; ++j) {
            const int key = k0 + j * RPR;
            int64_t at = key * ss;
            if constexpr (PAGED) {
              const int p = seq_page(a.kv, key), page = seq_same(tab[p - p0]);
              at = page * ps + (key - p * a.kv.page_size) * ss;
            }
            dma_x4_keep(base + at, (unsigned)(r * (int)ss + 16 * seq_chunk(c ^ (keys ? C::turn_k(j * RPR + r) : C::turn_v(j * RPR + r)), chunks)), dst + 1024 * j);
          }
          return;
        }
#pragma unroll
        for (int j = 0; j < S::NL; ++j) {
          const int i = j * 64 + seq_fresh<(C::RB > 128)>(lane), r = i / C::CB, c = (i - r * C::CB) ^ (keys ? C::turn_k(r) : C::turn_v(r));
          int key = k0 + r;
          key = key < ka ? ka : (key >= kb ? kb - 1 : key);
          int64_t at = key * ss;
          if constexpr (PAGED) {
            const int p = seq_page(a.kv, key);
            at = tab[p - p0] * ps + (key - p * a.kv.page_size) * ss;
          }
          dma_x4_from(base + at + 16 * seq_chunk(c, chunks), dst + 1024 * j);
          if (C::TIGHT) __builtin_amdgcn_sched_barrier(0);
        }
      };
      auto landed = [&](int h) __attribute__((always_inline)) {
        const int behind = halves - 1 - h;
        if (S::NB > 3 && behind >= 3) wait_vm<(S::NB > 3 ? 3 : 0) * S::NL>();
        else if (S::NB > 2 && behind >= 2) wait_vm<(S::NB > 2 ? 2 : 0) * S::NL>();
        else if (S::NB > 1 && behind >= 1) wait_vm<(S::NB > 1 ? 1 : 0) * S::NL>();
        else wait_vm<0>();
      };
      auto used = [&](int h) __attribute__((always_inline)) {
        if (h + S::NB < halves) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // half h is read
          issue(h + S::NB);
        }
      };
      for (int h = 0; h < S::NB && h < halves; ++h) issue(h);
      for (int t = c0; t < c1; ++t) {
        const int h = 2 * (t - c0), k0 = (u.t0 + t) * SEQ_STEP + 32 * wave;
        const bool some = k0 < kb && k0 + 32 > ka;
        f32x16 s;
        landed(h);
        if (some) {
          s = st.scores(ring + (unsigned)(h % S::NB * S::TB), 0, lane);
        }
        used(h);
        if (some) {
          if (k0 + 31 > first_place || (a.window > 0 && k0 <= last_place - a.window)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int back = place - (k0 + 8 * (i >> 2) + 4 * half + (i & 3));
              if (back < 0 || (a.window > 0 && back >= a.window)) s[i] = -INFINITY;
            }
          }
          float mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[i]);
          st.follow(xor32_max(mx), a.c);
          s = SeqState<T, DP>::held(st.weigh(s, a.c));
        }
        landed(h + 1);
        if (some) st.add(SeqState<T, DP>::taken(s), ring + (unsigned)((h + 1) % S::NB * S::TB), 0, lane);
        used(h + 1);
      }
    }
    // ---- the four waves' sums
    const float l = xor32_sum(st.l);
    if (half == 0) {
      ms[32 * wave + lane] = st.m;
      ls[32 * wave + lane] = l;
    }
    __syncthreads();  // everyone is done with the ring, and with the rows of the unit before
    if (threadIdx.x == 0) flag[4] = 0;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, ms[32 * w + (lane & 31)]);
    const float f = st.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((st.m - m) * a.c);
    float* part = (float*)smem_raw;
    if ((lane & 31) < n_rows) {
      float* mine = part + (32 * wave + (seq_fresh<C::TIGHT>(lane) & 31)) * S::PITCH + 4 * half;
#pragma unroll
      for (int n = 0; n < C::NMB; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          mine[32 * n + 8 * (i >> 2) + (i & 3)] = st.o[n][i] * f;
          if (C::TIGHT && i == 15) __builtin_amdgcn_sched_barrier(0);
        }
    }
    __syncthreads();
    const bool bad = PAGED && flag[1] != 0;
    const int cols = a.vchunks * C::E;
    const bool whole = !PAGED || (ta == 0 && tb == u.steps);
    const unsigned ws = (unsigned)((2 * share + (ta == 0 ? 1 : 0)) * 32 * (cols + 4));
    const __amdgpu_buffer_rsrc_t to = seq_parts_at(ra.ws);
    uint32_t odd = 0;
    for (int e = threadIdx.x; e < n_rows * (cols / 4); e += 256) {
      const int r = e / (cols / 4), d = 4 * (e - r * (cols / 4));
      float mr = -INFINITY, lr = 0.f;
      f32x4 o = f4_zero();
#pragma unroll
      for (int w = 0; w < 4; ++w) mr = fmaxf(mr, ms[32 * w + r]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float mw = ms[32 * w + r];
        lr += mw == -INFINITY ? ls[32 * w + r] : ls[32 * w + r] * __builtin_amdgcn_exp2f((mw - mr) * a.c);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += part[(32 * w + r) * S::PITCH + d + i];
      }
      if (bad) lr = NAN;
      if (whole) {
        const int tk = (r0 + r) / a.group, hd = head * a.group + r0 + r - tk * a.group;
        bool again = lr == 0.f && u.sp.length - u.sp.n + tk >= 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[i] = lr == 0.f ? 0.f : o[i] / lr;
          again |= !(fabsf(o[i]) < INFINITY);
        }
        odd |= (uint32_t)again << r;
        *(typename Tile<T>::quad*)(a.out + (u.sp.first + tk) * a.o_token + hd * a.o_head + d * (int)sizeof(T)) = to_quad<T>(o);
      } else {
        seq_give(to, ws + r * (cols + 4) + d, o);
        if (d == 0) seq_give(to, ws + r * (cols + 4) + cols, f32x4{mr, lr, 0.f, 0.f});
      }
    }
    if (PAGED && !whole) {
      int i0;
      const int parts = seq_parts(sc.total, n_shares, ahead + (int64_t)unit * places, places, i0);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every storing wave's stores are where the others look
      __syncthreads();
      if (threadIdx.x == 0) {
        flag[0] = __hip_atomic_fetch_add(&ra.brought[i0], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
        if (flag[0]) __hip_atomic_store(&ra.brought[i0], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      if (!__builtin_amdgcn_readfirstlane(flag[0])) continue;
      odd = seq_join<T>(ra, u, head, r0, n_rows, i0, parts, (float*)smem_raw, S::RING / 4, ls, (f32x4*)tab, wave, lane);
      tab_b = -1;
    }
    if (odd) __hip_atomic_fetch_or((uint32_t*)flag + 4, odd, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    __syncthreads();
    seq_finish<T, PAGED>(a, u, b, head, r0, (uint32_t)seq_same(flag[4]), wave, lane);
  }
}


template <class T, int DP>
__global__ __launch_bounds__(256, (SeqRows<T, DP>::LDS <= 80 * 1024 ? 2 : 1)) void k_seq_rows(const SeqRowsArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
  seq_rows<T, DP, true>(a, SeqRows<T, DP>::SHARES, blockIdx.x, smem_raw);
}

// Whole prompts that are few tiles of 128 rows: 32 rows a workgroup, and a quarter of their keys a wave.  grid (slots * kv_heads)
template <class T, int DP>
__global__ __launch_bounds__(256, (SeqRows<T, DP>::LDS <= 80 * 1024 ? 2 : 1)) void k_seq_blocks(const SeqArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
  seq_rows<T, DP, false>(SeqRowsArgs{a}, 0, blockIdx.x, smem_raw);
}

// ---- many rows, few tiles ----------------------------------------------------------------------------------------------------------
// Tiles of 128 rows over long keys that are too few for the chip - a portion of a prompt behind a long context - are cut along their
// keys: every tile into as many equal parts of at most T steps as it takes, with the least T whose parts are no more than the workgroups
// that fit on the chip at once; whole, where there are more tiles than those.  (Dealt like the units above, at borders wherever they fall, a workgroup has two parts to hand over and
// not one: 64 KB each, 8 x 256 tokens behind 1792 keys 138 us, 91 where no tile is cut.)  A part lies in the workspace as it lay in the
// registers ([wave][o ..., m, l][lane]), so that the workgroup that adds the parts, the last one to bring one, reads it lane by lane.
template <class T, int DP>
__device__ __forceinline__ void seq_tile_shares(const SeqRowsArgs& ra, int slots, int shares, int block, char* smem_raw) {
  typedef SeqTiles<T, DP> S;
  typedef SeqCfg<T, DP> C;
  int *tab = (int*)(smem_raw + S::RING), *flag = tab + SEQ_TAB, *pre = flag + 16;  // pre[i]: parts of a head ahead of slot i
  int* red = (int*)smem_raw;                                                       // sums of four waves, in the ring before it is used
  const SeqArgs& a = ra.s;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned lds0 = (unsigned)__builtin_amdgcn_readfirstlane((int)kh_lds_addr(smem_raw));
  // ---- steps of every slot, slot i a thread's of number i mod 256
  static_assert(S::MOST <= SEQ_TAB, "a sequence has a slot at least, so that the table has room for all offsets");
  for (int i = threadIdx.x; i < a.n_seqs; i += 256) tab[i] = a.offsets[i];
  __syncthreads();
  auto base_of = [&](int b) __attribute__((always_inline)) {
    const int o = tab[b];
    return (int)((int64_t)(o < 0 ? 0 : (o > a.n_tokens ? a.n_tokens : o)) * a.group / S::BM) + b;
  };
  constexpr int PER = S::MOST / 256;
  int steps[PER], all = 0, most = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = 256 * j + (int)threadIdx.x;
    steps[j] = 0;
    if (i >= slots) continue;
    int lo = 0, n = a.n_seqs;  // the last sequence whose base is at most i
    while (n > 1) {
      const int m = n / 2;
      if (base_of(lo + m) <= i) {
        lo += m;
        n -= m;
      } else {
        n = m;
      }
    }
    const SeqSpan sp = seq_span(a, lo);
    const int rows = sp.n * a.group, tiles = (rows + S::BM - 1) / S::BM, tile = tiles - 1 - (i - base_of(lo));
    if (rows <= 32 || tile < 0 || tile >= tiles) continue;
    const int r1 = tile * S::BM + S::BM - 1 < rows ? tile * S::BM + S::BM - 1 : rows - 1;
    const int q0 = sp.length - sp.n + tile * S::BM / a.group, q1 = sp.length - sp.n + r1 / a.group;
    const int k0 = a.window > 0 && q0 >= a.window ? q0 - a.window + 1 : 0;
    steps[j] = (q1 + S::BN) / S::BN - k0 / S::BN;
    if (q1 < 0 || steps[j] < 1) steps[j] = 1;  // no key at all: a step that writes the zeros
    all += steps[j] < 1 << 20 ? steps[j] : 1 << 20;  // in 32 bits; a lower bound is all it is for
    most = most > steps[j] ? most : steps[j];
  }
  // a sum over the workgroup, the same in every lane
  auto sum_of = [&](int x) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d);
    __syncthreads();
    if (lane == 0) red[wave] = x;
    __syncthreads();
    return seq_same(red[0] + red[1] + red[2] + red[3]);
  };
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_xor(most, d);
    most = most > y ? most : y;
  }
  if (lane == 0) red[4 + wave] = most;
  all = sum_of(all);
  if (all == 0) return;
  most = red[4] > red[5] ? red[4] : red[5];
  most = most > red[6] ? most : red[6];
  most = seq_same(most > red[7] ? most : red[7]);
  // the least T: at least an even share, at most the longest tile, which makes a part of every tile
  const int room = shares / a.kv_heads > 1 ? shares / a.kv_heads : 1;  // parts of a head
  int lo = (all + room - 1) / room, hi = most;
  lo = lo < S::LEAST ? S::LEAST : lo;
  hi = hi > lo ? hi : lo;
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    int n = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) n += (steps[j] + mid - 1) / mid;
    if (sum_of(n) <= room) hi = mid;
    else lo = mid + 1;
  }
  int cut[PER], before[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    int x = cut[j] = (steps[j] + lo - 1) / lo;
    if (256 * j < slots)
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x += y;
      }
    before[j] = x - cut[j];
    if (lane == 63) red[8 + 4 * j + wave] = x;
  }
  __syncthreads();
  int sum = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    for (int w = 0; w < 4; ++w) {
      if (w == wave) before[j] += sum;
      sum += red[8 + 4 * j + w];
    }
    const int i = 256 * j + (int)threadIdx.x;
    if (i < slots) pre[i] = before[j];
    if (i == slots - 1) pre[slots] = before[j] + cut[j];
  }
  __syncthreads();
  auto ahead = [&](int i) __attribute__((always_inline)) { return seq_same(pre[i]); };
  const int each = ahead(slots), parts_all = each * a.kv_heads;
  // ---- this workgroup's part, those of an XCD side by side, as their keys are
  const int side = (parts_all + 7) / 8, part = block % 8 * side + block / 8;
  if (block / 8 >= side || part >= parts_all) return;
  const int head = part / each, r = part - head * each;
  int slot = 0;
  for (int n = slots; n > 1;) {
    const int m = n / 2;
    if (ahead(slot + m) <= r) {
      slot += m;
      n -= m;
    } else {
      n = m;
    }
  }
  const int parts = ahead(slot + 1) - ahead(slot), p = r - ahead(slot);
  SeqTile s;
  if (!seq_tile<S::BM, S::BN, true>(a, slot, head, s, wave, lane)) return;  // offsets that do not ascend: none of the tile's parts runs
  if (threadIdx.x == 0) flag[1] = s.x.bad;
  SeqState<T, DP> st;
  st.load_q(a.q + (s.sp.first + s.token) * a.q_token + s.h * a.q_head, lane >> 5, a.kchunks);
  st.clear();
  const int n = s.t_hi > s.t_lo ? s.t_hi - s.t_lo : 0;
  __syncthreads();
  auto border = [&](int i) __attribute__((always_inline)) { return s.t_lo + (int)((int64_t)n * i / parts); };
  seq_tile_run<T, DP, true>(a, s, st, border(p), border(p + 1), lds0, tab, flag + 1, wave, lane);
  __syncthreads();
  float l = flag[1] ? -1.f : xor32_sum(st.l);  // -1: of a page that is none
  if (parts > 1) {
    const int blocks = (a.vchunks * C::E + 31) / 32, pitch = (16 * blocks + 4) * 64, first = part - p;  // pitch of a wave
    const __amdgpu_buffer_rsrc_t ws = seq_parts_at(ra.ws_tiles);
    auto at = [&](int i) __attribute__((always_inline)) { return (unsigned)(((first + i) * 4 + wave) * pitch + 4 * lane); };
    const unsigned to = at(p);
#pragma unroll
    for (int n = 0; n < C::NMB; ++n)
      if (n < blocks)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          seq_give(ws, to + (4 * n + i) * 256, f32x4{st.o[n][4 * i], st.o[n][4 * i + 1], st.o[n][4 * i + 2], st.o[n][4 * i + 3]});
        }
    seq_give(ws, to + 4 * blocks * 256, f32x4{st.m, l, 0.f, 0.f});
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every storing wave's stores are where the others look
    __syncthreads();
    if (threadIdx.x == 0) {
      flag[0] = __hip_atomic_fetch_add(&ra.brought_tiles[first], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
      if (flag[0]) __hip_atomic_store(&ra.brought_tiles[first], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!seq_same(flag[0])) return;
    float m = -INFINITY;
    for (int i = 0; i < parts; ++i) m = fmaxf(m, seq_take(ws, at(i) + 4 * blocks * 256)[0]);
    st.clear();
    bool none = false;
    l = 0.f;
    for (int i = 0; i < parts; ++i) {
      const unsigned from = at(i);
      const f32x4 ml = seq_take(ws, from + 4 * blocks * 256);
      const float f = ml[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml[0] - m) * a.c);
      none |= ml[1] < 0.f;
      l += ml[1] * f;
#pragma unroll
      for (int n = 0; n < C::NMB; ++n)
        if (n < blocks) {
          f32x4 v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = seq_take(ws, from + (4 * n + j) * 256);
#pragma unroll
          for (int j = 0; j < 16; ++j) st.o[n][j] = __builtin_fmaf(v[j / 4][j % 4], f, st.o[n][j]);
        }
    }
    if (none) l = -1.f;
  }
  seq_tile_write<T, DP, true>(a, s, st, l, l < 0.f, lane);
}

// Sequences of many rows and of few at once: half as many workgroups as the chip holds for the keys of the few between the first half
// for parts of tiles and the rest of those, so that both kinds are there from the start.  Two portions of a prompt among 30 single
// tokens, 32 heads of 64 over 4: 26 us (the portions alone 23, the single tokens alone 18), 34.5 with all for tiles ahead of as many
// for the few.  Either kind then has the other's registers, and the LDS of the larger: fp32 above 64 columns, where the rows' rings take 133 KB,
// one workgroup a CU for the tiles too, which alone would be two.  At heads of 256 each kind fills the registers, and they are
// launches of their own.
template <class T, int DP>
struct SeqMixed {
  static constexpr int LDS = SeqTiles<T, DP>::LDS_SHARES > SeqRows<T, DP>::LDS ? SeqTiles<T, DP>::LDS_SHARES : SeqRows<T, DP>::LDS;
  static constexpr int SHARES = LDS <= 80 * 1024 ? SEQ_SHARES : SEQ_SHARES / 2;  // of each
};
template <class T, int DP>
__global__ __launch_bounds__(256, (SeqMixed<T, DP>::LDS <= 80 * 1024 ? 2 : 1)) void k_seq_mixed(const SeqRowsArgs a, int slots) {
  extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
  constexpr int N = SeqMixed<T, DP>::SHARES, H = N / 2;
  const int i = blockIdx.x;
  if (i < H || i >= 2 * H) seq_tile_shares<T, DP>(a, slots, N, i < H ? i : i - H, smem_raw);
  else seq_rows<T, DP, true>(a, H, i - H, smem_raw);
}
template <class T, int DP>
__global__ __launch_bounds__(256, 1) void k_seq_tile_shares(const SeqRowsArgs a, int slots) {
  extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
  seq_tile_shares<T, DP>(a, slots, SeqMixed<T, DP>::SHARES, blockIdx.x, smem_raw);
}
}  // namespace khm
