// kh_rope_tokens.hip — rotary positions of many tokens, out of place or in place, and with keys and values written into a cache of
// pages.  No reference counterpart: its RoPE kernel rotates one token at a position of the host (cuda/rope_kernel.cu:104-170).
//
// Pair (a, b) of position p turns by the angle t = p f_i:  a' = m (a cos t - b sin t),  b' = m (a sin t + b cos t).
// The angle is formed in whole numbers: f_i / 2 pi is a 64-bit fraction of a turn, so p times it, modulo 2^64, is the angle modulo a
// turn with an error of |p| 2^-54 turns (the table's own: f_i has 53 bits), where fp32 loses p f_i 2^-24 radians: 0.004 at
// position 131072.  Its two highest bits, rounded, are the quadrant, and sine and cosine of what is left (at most an eighth of a
// turn either way) are the Taylor polynomials, cut where the rest is below 2^-25.
#include "kh_rows.h"
#include "kh_tile.h"

#include <math.h>

namespace khm {
namespace {

template <class T>
struct RopeArgs {
  const T *q, *k, *v;
  T *qo, *ko, *vo;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, qo_token, qo_head, ko_token, ko_head, vo_head;
  int64_t k_page, v_page, v_slot;  // of a cache: ko_token is then its k_slot
  const uint64_t* turns;
  const int32_t *positions, *slots;
  int heads, kv_heads, dim, vdim, rot, half, tokens;
  int n_pages, page_size;
  float magnitude;
};

__device__ __forceinline__ void cos_sin(uint64_t phase, float& c, float& s) {
  const uint64_t quad = (phase + (1ull << 61)) >> 62;  // mod 4
  const int32_t rest = (int32_t)((int64_t)(phase - (quad << 62)) >> 30);  // of 2^34 a turn, at most 2^31
  const float x = (float)rest * (float)(6.283185307179586 / 17179869184.0);
  const float z = x * x;
  float sn = 2.75573192e-6f, cs = -2.75573192e-7f;
  sn = __builtin_fmaf(sn, z, -1.98412698e-4f);
  sn = __builtin_fmaf(sn, z, 8.33333333e-3f);
  sn = __builtin_fmaf(sn, z, -1.66666667e-1f);
  sn = __builtin_fmaf(sn * z, x, x);
  cs = __builtin_fmaf(cs, z, 2.48015873e-5f);
  cs = __builtin_fmaf(cs, z, -1.38888889e-3f);
  cs = __builtin_fmaf(cs, z, 4.16666667e-2f);
  cs = __builtin_fmaf(cs, z, -0.5f);
  cs = __builtin_fmaf(cs, z, 1.0f);
  const float a = (quad & 1) ? sn : cs, b = (quad & 1) ? cs : sn;
  c = (quad == 1 || quad == 2) ? -a : a;
  s = (quad & 2) ? -b : b;
}

// Row of a cache that token t's keys and values go to; false: nowhere.
template <class T>
__device__ __forceinline__ bool place(const RopeArgs<T>& a, int t, int& page, int& slot) {
  const int s = a.slots[t];
  if (s < 0) return false;
  page = s / a.page_size;
  slot = s - page * a.page_size;
  return page < a.n_pages;
}

// One element, or one pair, a thread, with its angle formed for every head: rows and halves that are no whole vectors.  4096 tokens of 32 + 8 heads
// of 80 in bf16, 20 of them rotated: 32 us, by whole vectors (all 80) 17.  grid (tokens)
template <class T, bool STORE>
__global__ __launch_bounds__(256) void k_rope_pairs(const RopeArgs<T> a) {
  const int t = blockIdx.x;
  const int64_t pos = a.positions[t];
  int page = 0, slot = 0;
  const bool kept = !STORE || place(a, t, page, slot);
  const int per = a.rot / 2 + (a.dim - a.rot), both = (a.heads + a.kv_heads) * per;
  for (int w = threadIdx.x; w < both; w += 256) {
    const int h = w / per, i = w - h * per;
    const bool key = h >= a.heads;
    if (key && !kept) continue;
    const int kh = h - a.heads;
    const T* x = key ? a.k + t * a.k_token + kh * a.k_head : a.q + t * a.q_token + h * a.q_head;
    T* y = key ? (STORE ? a.ko + page * a.k_page + slot * a.ko_token + kh * a.ko_head : a.ko + t * a.ko_token + kh * a.ko_head)
               : a.qo + t * a.qo_token + h * a.qo_head;
    if (i >= a.rot / 2) {
      const int j = i + a.rot / 2;
      y[j] = x[j];
      continue;
    }
    const int j0 = a.half ? i : 2 * i, j1 = a.half ? i + a.rot / 2 : 2 * i + 1;
    float c, s;
    cos_sin((uint64_t)pos * a.turns[i], c, s);
    c *= a.magnitude;
    s *= a.magnitude;
    const float u = (float)x[j0], v = (float)x[j1];
    y[j0] = (T)(u * c - v * s);
    y[j1] = (T)(u * s + v * c);
  }
  if (STORE && kept)
    for (int w = threadIdx.x; w < a.kv_heads * a.vdim; w += 256) {
      const int h = w / a.vdim, j = w - h * a.vdim;
      a.vo[page * a.v_page + slot * a.v_slot + h * a.vo_head + j] = a.v[t * a.v_token + h * a.v_head + j];
    }
}

// The same by 16 bytes: a thread has two vectors of a head's row, E pairs in all - the vectors i of the two halves, or neighbours i - and
// keeps their cosines and sines for every head that it comes to, BATCH rows requested together.  HBM bounds it where the heads fill the workgroup:
// 8192 tokens of 32 + 32 heads of 128 with their values 83 us (4.8 TB/s), 4096 of 32 + 8 20.5; of 6 + 6 heads of 64, which are 48 threads' work,
// 11.3, where the bytes take 2.7: the start and end of 4096 workgroups.  grid (tokens)
template <class T, bool STORE>
__global__ __launch_bounds__(256) void k_rope_rows(const RopeArgs<T> a) {
  typedef typename Tile<T>::frag frag;
  constexpr int E = Tile<T>::N, BATCH = 4;
  const int t = blockIdx.x, per = a.dim / (2 * E), lead = (int)threadIdx.x / per, i = (int)threadIdx.x - lead * per, side = 256 / per;
  const int both = a.heads + a.kv_heads, turned = a.rot / (2 * E);
  const bool rotates = i < turned;
  // two vectors of a row, in elements
  const int c0 = E * (rotates ? (a.half ? i : 2 * i) : 2 * i), c1 = rotates && a.half ? c0 + a.rot / 2 : c0 + E;
  const int64_t pos = a.positions[t];
  int page = 0, slot = 0;
  const bool kept = !STORE || place(a, t, page, slot);
  auto from = [&](int r) __attribute__((always_inline)) {
    return r < a.heads ? a.q + t * a.q_token + r * a.q_head : a.k + t * a.k_token + (r - a.heads) * a.k_head;
  };
  auto to = [&](int r) __attribute__((always_inline)) {
    if (r < a.heads) return a.qo + t * a.qo_token + r * a.qo_head;
    return (STORE ? a.ko + page * a.k_page + slot * a.ko_token : a.ko + t * a.ko_token) + (r - a.heads) * a.ko_head;
  };
  frag x[BATCH], y[BATCH];
  auto load = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const int r = r0 + j * side;
      if (r < both) {
        const T* p = from(r);
        x[j] = *(const frag*)(p + c0);
        y[j] = *(const frag*)(p + c1);
      }
    }
  };
  const bool mine = lead < side;
  if (mine) load(lead);
  // values, as they are
  constexpr int VB = 2;
  frag v[VB];
  const int vper = STORE ? a.vdim / E : 1, values = STORE && kept ? a.kv_heads * vper : 0;
  auto vat = [&](int w, int& h) __attribute__((always_inline)) {
    h = w / vper;
    return E * (w - h * vper);
  };
  int h;
#pragma unroll
  for (int j = 0; j < VB; ++j)
    if ((int)threadIdx.x + 256 * j < values) {
      const int d = vat((int)threadIdx.x + 256 * j, h);
      v[j] = *(const frag*)(a.v + t * a.v_token + h * a.v_head + d);
    }
  float cs[E], sn[E];
  if (rotates)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      cos_sin((uint64_t)pos * a.turns[i * E + e], cs[e], sn[e]);
      cs[e] *= a.magnitude;
      sn[e] *= a.magnitude;
    }
  if (mine)
    for (int r0 = lead; r0 < both; r0 += BATCH * side) {
      if (r0 != lead) load(r0);
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const int r = r0 + j * side;
        if (r >= both || (r >= a.heads && !kept)) continue;
        frag u = x[j], w = y[j];
        if (rotates) {
          if (a.half) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const float p = (float)x[j][e], q = (float)y[j][e];
              u[e] = (T)(p * cs[e] - q * sn[e]);
              w[e] = (T)(p * sn[e] + q * cs[e]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const float p = (float)(e < E / 2 ? x[j][2 * e % E] : y[j][2 * e % E]), q = (float)(e < E / 2 ? x[j][(2 * e + 1) % E] : y[j][(2 * e + 1) % E]);
              const T lo = (T)(p * cs[e] - q * sn[e]), hi = (T)(p * sn[e] + q * cs[e]);
              if (e < E / 2) {
                u[2 * e % E] = lo;
                u[(2 * e + 1) % E] = hi;
              } else {
                w[2 * e % E] = lo;
                w[(2 * e + 1) % E] = hi;
              }
            }
          }
        }
        T* p = to(r);
        *(frag*)(p + c0) = u;
        *(frag*)(p + c1) = w;
      }
    }
  if (STORE) {
    T* vo = a.vo + page * a.v_page + slot * a.v_slot;
#pragma unroll
    for (int j = 0; j < VB; ++j)
      if ((int)threadIdx.x + 256 * j < values) {
        const int d = vat((int)threadIdx.x + 256 * j, h);
        *(frag*)(vo + h * a.vo_head + d) = v[j];
      }
    for (int w = (int)threadIdx.x + 256 * VB; w < values; w += 256) {
      const int d = vat(w, h);
      *(frag*)(vo + h * a.vo_head + d) = *(const frag*)(a.v + t * a.v_token + h * a.v_head + d);
    }
  }
}

template <class T, bool STORE>
int go(const RopeArgs<T>& a, hipStream_t s) {
  constexpr int E = Tile<T>::N;
  if (a.dim % (2 * E) == 0 && a.rot % (2 * E) == 0) hipLaunchKernelGGL((k_rope_rows<T, STORE>), dim3(a.tokens), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_rope_pairs<T, STORE>), dim3(a.tokens), dim3(256), 0, s, a);
  return kh_launch_status();
}

int check_rows(const kh_rope_rows* r, bool store) {
  if (!r || (r->dtype != KH_DTYPE_BF16 && r->dtype != KH_DTYPE_F32) || (r->mode != KH_ROPE_HALF && r->mode != KH_ROPE_INTERLEAVED) ||
      r->n_tokens < 0 || r->head_num <= 0 || r->kv_head_num <= 0 || r->head_num % r->kv_head_num || r->head_size <= 0 || r->rot_dim < 0 ||
      r->rot_dim % 2 || r->rot_dim > r->head_size || !(fabsf(r->magnitude) <= 3.4e38f))
    return KH_ERR_INVALID_ARG;
  const int e = r->dtype == KH_DTYPE_BF16 ? 2 : 4;
  if (!rows_whole(r->head_size, e) || r->head_size > 256 || r->n_tokens >= 1 << 24) return KH_ERR_UNSUPPORTED;  // a grid has 2^32 threads
  if (r->n_tokens == 0) return KH_OK;
  if ((r->rot_dim && !r->turns) || !r->positions || !r->q || !r->k || !r->q_out || (!store && !r->k_out) || !kh_aligned16(r->q) || !kh_aligned16(r->k) ||
      !kh_aligned16(r->q_out) || (!store && !kh_aligned16(r->k_out)) || !rows_whole(r->q_token, e) || !rows_whole(r->q_head, e) || !rows_whole(r->k_token, e) ||
      !rows_whole(r->k_head, e) || !rows_whole(r->qo_token, e) || !rows_whole(r->qo_head, e) || (!store && (!rows_whole(r->ko_token, e) || !rows_whole(r->ko_head, e))))
    return KH_ERR_INVALID_ARG;
  // a result has a place of its own
  if ((!store && r->q_out == r->k_out) || !rows_apart({r->n_tokens, r->head_num}, {r->qo_token, r->qo_head}, r->head_size) ||
      (!store && !rows_apart({r->n_tokens, r->kv_head_num}, {r->ko_token, r->ko_head}, r->head_size)))
    return KH_ERR_INVALID_ARG;
  // in place: a row is written where it was read
  auto moved = [&](int64_t token, int64_t head, int64_t o_token, int64_t o_head, int heads) {
    return (token != o_token && r->n_tokens > 1) || (head != o_head && heads > 1);
  };
  if ((r->q == r->q_out && moved(r->q_token, r->q_head, r->qo_token, r->qo_head, r->head_num)) ||
      (!store && r->k == r->k_out && moved(r->k_token, r->k_head, r->ko_token, r->ko_head, r->kv_head_num)))
    return KH_ERR_INVALID_ARG;
  return KH_OK;
}

template <class T>
RopeArgs<T> args_of(const kh_rope_rows* r) {
  RopeArgs<T> a{};
  a.q = (const T*)r->q;
  a.k = (const T*)r->k;
  a.qo = (T*)r->q_out;
  a.ko = (T*)r->k_out;
  a.q_token = r->q_token;
  a.q_head = r->q_head;
  a.k_token = r->k_token;
  a.k_head = r->k_head;
  a.qo_token = r->qo_token;
  a.qo_head = r->qo_head;
  a.ko_token = r->ko_token;
  a.ko_head = r->ko_head;
  a.turns = r->turns;
  a.positions = r->positions;
  a.heads = r->head_num;
  a.kv_heads = r->kv_head_num;
  a.dim = r->head_size;
  a.rot = r->rot_dim;
  a.half = r->mode == KH_ROPE_HALF;
  a.tokens = r->n_tokens;
  a.magnitude = r->magnitude;
  return a;
}

template <class T>
int store(const kh_rope_rows* r, const void* v, int64_t v_token, int64_t v_head, int value_size, const kh_page_cache* c,
          const int32_t* slots, hipStream_t s) {
  RopeArgs<T> a = args_of<T>(r);
  a.v = (const T*)v;
  a.v_token = v_token;
  a.v_head = v_head;
  a.vdim = value_size;
  a.ko = (T*)c->k;
  a.vo = (T*)c->v;
  a.k_page = c->k_page;
  a.ko_token = c->k_slot;
  a.ko_head = c->k_head;
  a.v_page = c->v_page;
  a.v_slot = c->v_slot;
  a.vo_head = c->v_head;
  a.slots = slots;
  a.n_pages = c->n_pages;
  a.page_size = c->page_size;
  return go<T, true>(a, s);
}
}  // namespace
}  // namespace khm

extern "C" int kh_rope_turns(int32_t rot_dim, double theta, const kh_rope_scaling* c, uint64_t* h_turns, float* h_magnitude) {
  if (rot_dim < 0 || rot_dim % 2 || rot_dim > 256 || !(theta > 0) || !(theta < 1e300) || (rot_dim && !h_turns) || !h_magnitude) return KH_ERR_INVALID_ARG;
  const int kind = c ? c->kind : KH_ROPE_SCALE_NONE;
  if (kind < KH_ROPE_SCALE_NONE || kind > KH_ROPE_SCALE_RAMP) return KH_ERR_INVALID_ARG;
  if (kind != KH_ROPE_SCALE_NONE && (!(c->factor > 0) || !(c->factor < 1e300))) return KH_ERR_INVALID_ARG;
  if (kind == KH_ROPE_SCALE_BANDS && (!(c->original > 0) || !(c->low > 0) || !(c->high > c->low))) return KH_ERR_INVALID_ARG;
  if (kind == KH_ROPE_SCALE_RAMP && (!(c->original > 0) || !(c->slow > 0) || !(c->fast > c->slow) || !(theta > 1) || !(c->magnitude >= 0)))
    return KH_ERR_INVALID_ARG;
  const double two_pi = 6.283185307179586476925;
  double lo = 0, hi = 0;
  *h_magnitude = 1.f;
  if (kind == KH_ROPE_SCALE_RAMP) {
    auto pair = [&](double turns) { return rot_dim * log(c->original / (turns * two_pi)) / (2 * log(theta)); };
    lo = floor(pair(c->fast));
    hi = ceil(pair(c->slow));
    lo = lo > 0 ? lo : 0;
    hi = hi < rot_dim - 1 ? hi : rot_dim - 1;
    *h_magnitude = (float)(c->magnitude > 0 ? c->magnitude : (c->factor > 1 ? 0.1 * log(c->factor) + 1.0 : 1.0));
    if (!(*h_magnitude < INFINITY)) return KH_ERR_INVALID_ARG;
  }
  for (int i = 0; i < rot_dim / 2; ++i) {
    double f = pow(theta, -2.0 * i / rot_dim);
    if (kind == KH_ROPE_SCALE_LINEAR) f /= c->factor;
    if (kind == KH_ROPE_SCALE_BANDS) {
      double keep = (c->original * f / two_pi - c->low) / (c->high - c->low);
      keep = keep < 0 ? 0 : (keep > 1 ? 1 : keep);
      f = f * keep + f / c->factor * (1 - keep);
    }
    if (kind == KH_ROPE_SCALE_RAMP) {
      const double width = hi - lo > 0.001 ? hi - lo : 0.001;
      double g = (i - lo) / width;
      g = g < 0 ? 0 : (g > 1 ? 1 : g);
      f = f / c->factor * g + f * (1 - g);
    }
    double turn = f / two_pi;
    if (!(turn < INFINITY)) return KH_ERR_INVALID_ARG;  // theta, factor or a border beyond what a frequency holds
    turn -= floor(turn);  // a frequency may be of more than a turn
    h_turns[i] = (uint64_t)ldexp(turn, 64);
  }
  return KH_OK;
}

extern "C" int kh_rope_tokens(const kh_rope_rows* r, void* stream) {
  const int rc = khm::check_rows(r, false);
  if (rc != KH_OK || r->n_tokens == 0) return rc;
  return r->dtype == KH_DTYPE_BF16 ? khm::go<khm::bf16, false>(khm::args_of<khm::bf16>(r), (hipStream_t)stream)
                                   : khm::go<float, false>(khm::args_of<float>(r), (hipStream_t)stream);
}

extern "C" int kh_rope_store(const kh_rope_rows* r, const void* v, int64_t v_token, int64_t v_head, int32_t value_size,
                             const kh_page_cache* c, const int32_t* slots, void* stream) {
  const int rc = khm::check_rows(r, true);
  if (rc != KH_OK) return rc;
  const int e = r->dtype == KH_DTYPE_BF16 ? 2 : 4;
  if (value_size <= 0) return KH_ERR_INVALID_ARG;
  if (!khm::rows_whole(value_size, e) || value_size > 256) return KH_ERR_UNSUPPORTED;
  if (r->n_tokens == 0) return KH_OK;
  if (!v || !c || !slots || !c->k || !c->v || c->n_pages <= 0 || c->page_size <= 0 || !kh_aligned16(v) || !kh_aligned16(c->k) ||
      !kh_aligned16(c->v) || !khm::rows_whole(v_token, e) || !khm::rows_whole(v_head, e) || !khm::rows_whole(c->k_page, e) || !khm::rows_whole(c->k_slot, e) ||
      !khm::rows_whole(c->k_head, e) || !khm::rows_whole(c->v_page, e) || !khm::rows_whole(c->v_slot, e) || !khm::rows_whole(c->v_head, e) ||
      c->k == c->v || !khm::rows_apart({c->n_pages, c->page_size, r->kv_head_num}, {c->k_page, c->k_slot, c->k_head}, r->head_size) ||
      !khm::rows_apart({c->n_pages, c->page_size, r->kv_head_num}, {c->v_page, c->v_slot, c->v_head}, value_size))
    return KH_ERR_INVALID_ARG;
  return r->dtype == KH_DTYPE_BF16 ? khm::store<khm::bf16>(r, v, v_token, v_head, value_size, c, slots, (hipStream_t)stream)
                                   : khm::store<float>(r, v, v_token, v_head, value_size, c, slots, (hipStream_t)stream);
}
