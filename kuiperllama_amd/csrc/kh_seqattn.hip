// kh_seqattn.hip — attention of many sequences' tokens: checks and launches (kernels in kh_seqattn.h).
#include "kh_rows.h"
#include "kh_seqattn.h"

#include <limits.h>

namespace khm {
namespace {

constexpr float LOG2E = 1.4426950408889634f;

// Common checks; *todo = 0: nothing to do.
int check_rows(const kh_attn_rows* r, int* esize, int* todo) {
  *todo = 0;
  if (!r || (r->dtype != KH_DTYPE_BF16 && r->dtype != KH_DTYPE_F32) || r->n_tokens < 0 || r->n_seqs < 0 || r->head_num <= 0 ||
      r->kv_head_num <= 0 || r->head_num % r->kv_head_num || r->head_size <= 0 || r->value_size <= 0 || !(r->scale > 0.f) ||
      !(r->scale * LOG2E < INFINITY))
    return KH_ERR_INVALID_ARG;
  const int e = *esize = r->dtype == KH_DTYPE_BF16 ? 2 : 4;
  if (!rows_whole(r->head_size, e) || !rows_whole(r->value_size, e) || r->head_size > 256 || r->value_size > 256) return KH_ERR_UNSUPPORTED;
  // rows of a sequence are counted in 32 bits, and a grid has 2^32 threads
  if ((int64_t)r->n_tokens * r->head_num > INT_MAX / 2 || (int64_t)r->n_tokens * r->head_num / 128 + (int64_t)r->n_seqs * r->kv_head_num >= 1 << 24)
    return KH_ERR_UNSUPPORTED;
  if (r->n_tokens == 0 || r->n_seqs == 0) return KH_OK;
  if (!r->offsets || !r->q || !r->out || r->q == r->out || !kh_aligned16(r->q) || !kh_aligned16(r->out) || !rows_whole(r->q_token, e) || !rows_whole(r->q_head, e) ||
      !rows_whole(r->o_token, e) || !rows_whole(r->o_head, e) ||
      !rows_apart({r->n_tokens, r->head_num}, {r->o_token, r->o_head}, r->value_size))
    return KH_ERR_INVALID_ARG;
  *todo = 1;
  return KH_OK;
}

SeqArgs args_of(const kh_attn_rows* r, int e) {
  SeqArgs a{};
  a.q = (const char*)r->q;
  a.out = (char*)r->out;
  a.q_token = r->q_token * e;
  a.q_head = r->q_head * e;
  a.o_token = r->o_token * e;
  a.o_head = r->o_head * e;
  a.offsets = r->offsets;
  a.n_tokens = r->n_tokens;
  a.n_seqs = r->n_seqs;
  a.heads = r->head_num;
  a.kv_heads = r->kv_head_num;
  a.group = r->head_num / r->kv_head_num;
  a.kchunks = r->head_size * e / 16;
  a.vchunks = r->value_size * e / 16;
  // places and lengths stay below 2^30 either way: a window of more holds everything, and a place less one of no more has room in 32 bits
  a.window = r->window > INT_MAX / 2 ? 0 : r->window;
  a.c = r->scale * LOG2E;
  return a;
}

template <class K, class... A>
int launch(K kern, dim3 grid, int lds, hipStream_t s, const A&... a) {
  if (lds > 64 * 1024) KH_CHECK_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  hipLaunchKernelGGL(kern, grid, dim3(256), lds, s, a...);
  return kh_launch_status();
}

// How a call is launched: whole prompts, in tiles of 128 rows or of 32; over pages, few rows alone where no sequence has more than 32, else
// tiles of rows and, at once or behind them, the rows of the sequences that have few.
enum How { PACKED, FEW, ANY };
template <class T, int DP>
int go(SeqRowsArgs a, How how, hipStream_t s) {
  typedef SeqTiles<T, DP> S;
  typedef SeqRows<T, DP> R;
  typedef SeqMixed<T, DP> M;
  constexpr int CB = SeqCfg<T, DP>::CB;
  const SeqKv& kv = a.s.kv;
  auto near = [](int64_t stride) { return stride >= 0 && stride < 1 << 24; };  // 64 rows apart in 32 bits
  a.s.kv.plain = near(kv.k_slot) && near(kv.v_slot) && (!kv.pages || kv.page_size % (64 / CB) == 0);
  a.all = how == FEW;
  if (how == FEW) return launch(k_seq_rows<T, DP>, dim3(R::SHARES), R::LDS, s, a);
  const int64_t slots = (int64_t)a.s.n_tokens * a.s.group / S::BM + a.s.n_seqs;
  const dim3 grid((unsigned)(slots * a.s.kv_heads));
  if (how == PACKED) {
    // Tiles that are too few wait for the longest of them, which workgroups of 32 rows and a quarter of the keys a wave have done in a fourth
    // of the time, for four times the requests.  us, blocks and tiles of 128: bf16, heads of 128, 14 over 2, 1000 tokens (109 tiles) 20, 29;
    // 2000 (218) 46, 57; 32 over 8, 1024 (256) 37, 33; 250 of 14 over 2 12, 11.  fp32, 14 over 2, 1000 tokens 64, 130; 4000 (437) 625,
    // 501, of 64 235, 286; 8 x 64 of 32 over 32 34, 22.
    const bool fp32 = sizeof(T) == 4;
    const int most = fp32 ? (DP <= 64 ? 512 : 256) : 224;
    if ((int64_t)a.s.n_tokens * a.s.group / S::BM * a.s.kv_heads <= most && a.s.n_tokens / a.s.n_seqs >= (fp32 ? 192 : 384)) {
      const int64_t blocks = (int64_t)a.s.n_tokens * a.s.group / 32 + a.s.n_seqs;
      return launch(k_seq_blocks<T, DP>, dim3((unsigned)(blocks * a.s.kv_heads)), R::LDS, s, a.s);
    }
    return launch(k_seq_tiles<T, DP, false>, grid, S::LDS_PACKED, s, a.s);
  }
  // Tiles that are fewer than the workgroups the chip holds are cut along their keys (136 tiles of 512 tokens behind 16384 keys: 345 us,
  // 1214 whole; 16 of 64 behind 4096: 33, 81); as many or more are left whole (512 of 2048 tokens behind 8192: 290 us, 333 with
  // cuts).  How many there are depends on the offsets: by the tokens no more than these and one for each sequence.
  unsigned parts = 0;
  if (slots <= S::MOST && (int64_t)a.s.n_tokens * a.s.group / S::BM * a.s.kv_heads < M::SHARES) {
    parts = ((unsigned)(slots * a.s.kv_heads > M::SHARES ? slots * a.s.kv_heads : M::SHARES) + 7) / 8 * 8;
    a.brought_tiles = a.brought + SEQ_SHARES;
    a.ws_tiles = a.ws + (size_t)2 * SEQ_SHARES * 32 * (a.s.vchunks * (16 / (int)sizeof(T)) + 4);
    if constexpr (DP <= 128) return launch(k_seq_mixed<T, DP>, dim3(M::SHARES / 2 + parts), M::LDS, s, a, (int)slots);
  }
  int rc;
  if (DP > 128 && a.ws_tiles) rc = launch(k_seq_tile_shares<T, 256>, dim3(parts), S::LDS_SHARES, s, a, (int)slots);
  else rc = launch(k_seq_tiles<T, DP, true>, grid, S::LDS_PAGED, s, a.s);
  return rc != KH_OK ? rc : launch(k_seq_rows<T, DP>, dim3(R::SHARES), R::LDS, s, a);
}

int go(const SeqRowsArgs& a, int e, How how, hipStream_t s) {
  const int most = (a.s.kchunks > a.s.vchunks ? a.s.kchunks : a.s.vchunks) * 16 / e;
  if (e == 2) return most <= 64 ? go<bf16, 64>(a, how, s) : most <= 96 ? go<bf16, 96>(a, how, s) : (most <= 128 ? go<bf16, 128>(a, how, s) : go<bf16, 256>(a, how, s));
  return most <= 64 ? go<float, 64>(a, how, s) : most <= 96 ? go<float, 96>(a, how, s) : (most <= 128 ? go<float, 128>(a, how, s) : go<float, 256>(a, how, s));
}
}  // namespace
}  // namespace khm

extern "C" int kh_attn_packed(const kh_attn_rows* r, const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token,
                              int64_t v_head, void* stream) {
  int e, todo;
  const int rc = khm::check_rows(r, &e, &todo);
  if (rc != KH_OK || !todo) return rc;
  if (!k || !v || k == r->out || v == r->out || !kh_aligned16(k) || !kh_aligned16(v) || !khm::rows_whole(k_token, e) || !khm::rows_whole(k_head, e) || !khm::rows_whole(v_token, e) ||
      !khm::rows_whole(v_head, e))
    return KH_ERR_INVALID_ARG;
  khm::SeqRowsArgs ra{khm::args_of(r, e)};
  khm::SeqArgs& a = ra.s;
  a.kv.k = (const char*)k;
  a.kv.v = (const char*)v;
  a.kv.k_slot = k_token * e;
  a.kv.k_head = k_head * e;
  a.kv.v_slot = v_token * e;
  a.kv.v_head = v_head * e;
  return khm::go(ra, e, khm::PACKED, (hipStream_t)stream);
}

extern "C" int64_t kh_attn_paged_workspace_bytes(int32_t head_num, int32_t kv_head_num, int32_t value_size, int32_t n_tokens) {
  if (head_num <= 0 || kv_head_num <= 0 || head_num % kv_head_num || value_size <= 0 || n_tokens < 0) return KH_ERR_INVALID_ARG;
  // counters, two parts of 32 rows a share, and one of 128 rows as four waves hold them where a call can have as many
  const bool tiles = (int64_t)n_tokens * (head_num / kv_head_num) > 32;
  return 4 * (2 * khm::SEQ_SHARES + 2 * khm::SEQ_SHARES * 32 * ((int64_t)value_size + 4) +
              (tiles ? khm::SEQ_SHARES * (int64_t)4 * 64 * (16 * ((value_size + 31) / 32) + 4) : 0));
}

extern "C" int kh_attn_paged(const kh_attn_rows* r, const kh_page_cache* c, const int32_t* pages, int64_t table_stride,
                             int32_t table_width, const int32_t* lengths, int32_t max_new, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  int e, todo;
  const int rc = khm::check_rows(r, &e, &todo);
  if (rc != KH_OK) return rc;
  if (!c || c->n_pages <= 0 || c->page_size <= 0 || c->page_size > 1 << 20 || table_width <= 0 || table_stride < 0 || max_new < 0)
    return KH_ERR_INVALID_ARG;
  if (!todo) return KH_OK;
  if (!c->k || !c->v || c->k == r->out || c->v == r->out || !pages || !lengths || !kh_aligned16(c->k) || !kh_aligned16(c->v) || !khm::rows_whole(c->k_page, e) ||
      !khm::rows_whole(c->k_slot, e) || !khm::rows_whole(c->k_head, e) || !khm::rows_whole(c->v_page, e) || !khm::rows_whole(c->v_slot, e) ||
      !khm::rows_whole(c->v_head, e) || !workspace || !kh_aligned16(workspace) ||
      workspace_bytes < kh_attn_paged_workspace_bytes(r->head_num, r->kv_head_num, r->value_size, r->n_tokens))
    return KH_ERR_INVALID_ARG;
  khm::SeqRowsArgs ra{khm::args_of(r, e), (int*)workspace, (float*)workspace + 2 * khm::SEQ_SHARES};
  khm::SeqArgs& a = ra.s;
  a.kv.k = (const char*)c->k;
  a.kv.v = (const char*)c->v;
  a.kv.k_page = c->k_page * e;
  a.kv.k_slot = c->k_slot * e;
  a.kv.k_head = c->k_head * e;
  a.kv.v_page = c->v_page * e;
  a.kv.v_slot = c->v_slot * e;
  a.kv.v_head = c->v_head * e;
  a.kv.pages = pages;
  a.kv.table_stride = table_stride;
  a.kv.most = (int64_t)table_width * c->page_size < INT_MAX / 2 ? table_width * c->page_size : INT_MAX / 2;
  a.kv.n_pages = c->n_pages;
  a.kv.page_size = c->page_size;
  // for d = page_size >= 2, 2^(b-1) < d <= 2^b: floor(2^(31+b) / d) + 1 is too large by at most 1, so its product with n < 2^31 by
  // less than 2^(31+b) / d, and the quotient is exact
  int bits = 0;
  while ((1 << bits) < c->page_size) ++bits;
  a.kv.magic = c->page_size == 1 ? 0 : (uint32_t)((1ull << (31 + bits)) / (uint64_t)c->page_size + 1);
  a.kv.shift = bits - 1;
  a.kv.lengths = lengths;
  const int64_t most = (int64_t)(max_new && max_new < r->n_tokens ? max_new : r->n_tokens) * a.group;
  return khm::go(ra, e, most <= 32 ? khm::FEW : khm::ANY, (hipStream_t)stream);
}
