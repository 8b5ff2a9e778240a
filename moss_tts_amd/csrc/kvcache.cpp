// C ABI of the drafted-token operators (include/mtts.h): argument checks and launches.
#include <algorithm>
#include <cmath>

#include "engine_internal.h"
#include "kvq.h"

using namespace mtts;

namespace {

constexpr int KV_SLOTS_MAX = 1 << 25;  // (lane offsets into a cache row are 32 bits of bytes; tile counts round up in 32 bits)

bool view_of(const mtts_kv_cache* c, KvView* v, const char** why) {
  *why = nullptr;
  if (!c || !c->k || !c->v) *why = "cache required";
  else if (c->type != KV_BF16 && c->type != KV_E4M3 && c->type != KV_INT8) *why = "cache type is bf16, e4m3 or int8";
  else if (c->type != KV_BF16 && (!c->k_scale || !c->v_scale)) *why = "an 8-bit cache needs its scales";
  else if (c->rows < 1 || c->n_kv < 1 || c->slots < 32 || c->slots % 32 || c->slots >= KV_SLOTS_MAX)
    *why = "cache rows, heads and slots (a multiple of 32, below 2^25)";
  else if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 15)
    *why = "cache pointers are 16-byte aligned";
  if (*why) return false;
  *v = KvView{c->k, c->v, c->k_scale, c->v_scale, c->type, c->rows, c->n_kv, c->head_dim, c->slots};
  return true;
}
bool dim_ok(int D) { return D == 32 || D == 64 || D == 128; }

bool rope_of(const mtts_rope* r, int D, RopeView* v) {
  *v = RopeView{nullptr, 0, 0, 1.f};
  if (!r || r->rotary_dim == 0) return true;
  if (r->rotary_dim < 0 || r->rotary_dim % 2 || r->rotary_dim > D || !r->turns) return false;
  *v = RopeView{r->turns, r->rotary_dim, r->interleaved != 0, r->factor};
  return true;
}

// n rows of m pieces of d elements, at strides ld and hs: no two meet (one side's run lies within a stride of
// the other)
bool apart(int n, size_t ld, int m, size_t hs, size_t d) {
  if (n > 1 && m > 1) return (hs >= d && ld >= (m - 1) * hs + d) || (ld >= d && hs >= (n - 1) * ld + d);
  return (n < 2 || ld >= d) && (m < 2 || hs >= d);
}


// The bytes of a tensor argument: n[0] x n[1] runs of `run` bytes, s[i] bytes apart.
struct Runs {
  uintptr_t at;
  int64_t run, s[2], n[2];
  Runs(const void* p, int n0, size_t s0, int n1, size_t s1, int64_t d)  // in elements of 2 bytes
      : at((uintptr_t)p), run(2 * d), s{2 * (int64_t)s0, 2 * (int64_t)s1}, n{n0, n1} {
    // runs that touch or lie in one another are one
    for (int again = 0; again < 2; ++again)
      for (int i = 0; i < 2; ++i)
        if (s[i] <= run || n[i] < 2) {
          run += (n[i] - 1) * (n[i] < 2 ? 0 : s[i]);
          n[i] = 1;
          s[i] = 0;
        }
  }
  int64_t end() const { return (n[0] - 1) * s[0] + (n[1] - 1) * s[1] + run; }
};
// whether lo < c + sum of s t < hi for some t, from t.lo to t.hi each; strides in falling order
struct Term {
  int64_t s, lo, hi;
};
bool hits(const Term* t, int n, int64_t c, int64_t lo, int64_t hi) {
  if (n == 0) return lo < c && c < hi;
  int64_t least = c, most = c;
  for (int i = 1; i < n; ++i) {
    least += t[i].s * t[i].lo;
    most += t[i].s * t[i].hi;
  }
  const auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
  const int64_t first = std::max(t->lo, -floor_div(most - lo - 1, t->s)), last = std::min(t->hi, floor_div(hi - 1 - least, t->s));
  for (int64_t x = first; x <= last; ++x)
    if (hits(t + 1, n - 1, c + x * t->s, lo, hi)) return true;
  return false;
}
// whether two arguments share a byte: at once if their extents do not meet (nearly every call), else by the
// differences of their runs' places
bool share(const Runs& a, const Runs& b) {
  const int64_t c = (int64_t)(b.at - a.at);
  if (c >= a.end() || -c >= b.end()) return false;
  Term t[4];
  int n = 0;
  const auto add = [&](int64_t s, int64_t lo, int64_t hi) {
    if (lo == hi) return;
    for (int i = 0; i < n; ++i)
      if (t[i].s == s) {
        t[i].lo += lo;
        t[i].hi += hi;
        return;
      }
    t[n++] = Term{s, lo, hi};
  };
  for (int i = 0; i < 2; ++i) add(a.s[i], 1 - a.n[i], 0);
  for (int i = 0; i < 2; ++i) add(b.s[i], 0, b.n[i] - 1);
  std::sort(t, t + n, [](const Term& x, const Term& y) { return x.s > y.s; });
  return hits(t, n, c, -b.run, a.run);
}

}  // namespace

#define KV_CACHE(c, v)                                            \
  KvView v;                                                       \
  const char* why_;                                               \
  if (!view_of(c, &v, &why_)) return fail(MTTS_E_INVALID, why_);  \
  if (!dim_ok(v.D)) return fail(MTTS_E_UNSUPPORTED, "head_dim is 32, 64 or 128")

extern "C" size_t mtts_kv_bytes(int type, int rows, int n_kv, int head_dim, int slots) {
  return (size_t)rows * n_kv * slots * head_dim * (type == KV_BF16 ? 2 : 1);
}

extern "C" int mtts_rope_turns(double theta, int rot, const mtts_rope_scaling* sc, double* turns, float* factor) {
  if (!turns || !factor || rot < 2 || rot % 2 || !(theta > 1.0) || !std::isfinite(theta))
    return fail(MTTS_E_INVALID, "rope: even rotary dim, base > 1");
  const int kind = sc ? sc->kind : MTTS_ROPE_DEFAULT;
  const double two_pi = 6.283185307179586476925286766559;
  if (kind < MTTS_ROPE_DEFAULT || kind > MTTS_ROPE_LLAMA3) return fail(MTTS_E_INVALID, "rope: unknown scaling");
  if (kind != MTTS_ROPE_DEFAULT && !(sc->factor >= 1.0 && std::isfinite(sc->factor)))
    return fail(MTTS_E_INVALID, "rope: a finite scaling factor >= 1");
  if ((kind == MTTS_ROPE_YARN || kind == MTTS_ROPE_LLAMA3) &&
      !(sc->original_max_position > 0 && std::isfinite(sc->original_max_position)))
    return fail(MTTS_E_INVALID, "rope: the original length is required");
  if (kind == MTTS_ROPE_YARN && !(sc->beta_slow > 0 && sc->beta_fast >= sc->beta_slow && std::isfinite(sc->beta_fast)))
    return fail(MTTS_E_INVALID, "rope: beta_fast >= beta_slow > 0");
  if (kind == MTTS_ROPE_YARN && !std::isfinite(sc->attention_factor))
    return fail(MTTS_E_INVALID, "rope: a finite attention factor");
  if (kind == MTTS_ROPE_LLAMA3 && !(sc->high_freq > sc->low_freq && std::isfinite(sc->low_freq) && std::isfinite(sc->high_freq)))
    return fail(MTTS_E_INVALID, "rope: high_freq > low_freq");
  if (kind == MTTS_ROPE_NTK && rot == 2) return fail(MTTS_E_INVALID, "rope: ntk scaling needs more than one pair");
  *factor = 1.f;
  const double base = kind == MTTS_ROPE_NTK ? theta * std::pow(sc->factor, rot / (rot - 2.0)) : theta;
  double lo = 0, hi = 0;
  if (kind == MTTS_ROPE_YARN) {
    // the pair that makes beta turns over the original length
    auto pair_of = [&](double beta) {
      return rot * std::log(sc->original_max_position / (beta * two_pi)) / (2.0 * std::log(theta));
    };
    lo = std::fmax(0.0, std::floor(pair_of(sc->beta_fast)));
    hi = std::fmin(rot - 1.0, std::ceil(pair_of(sc->beta_slow)));
    *factor = (float)(sc->attention_factor > 0 ? sc->attention_factor : 0.1 * std::log(sc->factor) + 1.0);
  }
  for (int i = 0; i < rot / 2; ++i) {
    double f = std::pow(base, -2.0 * i / rot);
    if (kind == MTTS_ROPE_LINEAR) f /= sc->factor;
    else if (kind == MTTS_ROPE_YARN) {
      const double ramp = std::fmin(1.0, std::fmax(0.0, (i - lo) / std::fmax(hi - lo, 0.001)));
      f = ramp * f / sc->factor + (1.0 - ramp) * f;
    } else if (kind == MTTS_ROPE_LLAMA3) {
      const double turns_old = sc->original_max_position * f / two_pi;
      const double keep = std::fmin(1.0, std::fmax(0.0, (turns_old - sc->low_freq) / (sc->high_freq - sc->low_freq)));
      f = (1.0 - keep) * f / sc->factor + keep * f;
    }
    turns[i] = f / two_pi;
  }
  return 0;
}

extern "C" int mtts_k_rope(const uint16_t* x, size_t ldx, size_t hsx, uint16_t* y, size_t ldy, size_t hsy,
                           const int32_t* pos, int M, int H, int D, const mtts_rope* rope, void* stream) {
  if (M < 0 || H < 0 || D < 2 || D % 2) return fail(MTTS_E_INVALID, "rope: bad sizes");
  if (M == 0 || H == 0) return 0;
  RopeArgs a{x, y, ldx, hsx, ldy, hsy, pos, M, H, D, {}};
  if (!x || !y || !pos || !rope) return fail(MTTS_E_INVALID, "rope: bad arguments");
  if (!apart(M, ldy, H, hsy, D)) return fail(MTTS_E_INVALID, "rope: the output's heads overlap");
  // (a wave rotates a head in its registers: in place it is read before it is written; any other head that is
  // shared would be read by one wave before or after another has written it)
  const bool in_place = x == y && (M == 1 || ldx == ldy) && (H == 1 || hsx == hsy);
  if (!in_place && share(Runs(x, M, ldx, H, hsx, D), Runs(y, M, ldy, H, hsy, D)))
    return fail(MTTS_E_INVALID, "rope: the output overlaps the input (in place is fine, with its strides)");
  if (!rope_of(rope, D, &a.r)) return fail(MTTS_E_INVALID, "rope: bad arguments");
  HIPCHK(rope_apply(a, (hipStream_t)stream));
  return 0;
}

extern "C" int mtts_k_kv_append(const mtts_kv_cache* cache, const uint16_t* q, size_t ldq, const uint16_t* k, size_t ldk,
                                const uint16_t* v, size_t ldv, uint16_t* q_out, size_t ldqo, int n_heads,
                                const uint16_t* qn, const uint16_t* kn, float eps, const mtts_rope* rope,
                                const int32_t* pos, const int32_t* start, const int32_t* counts, int B, int S,
                                void* stream) {
  KV_CACHE(cache, c);
  if (B < 0 || B > c.rows || S < 0) return fail(MTTS_E_INVALID, "append: more rows than the cache has");
  if (B == 0 || S == 0) return 0;
  if (!k || !v || !start || (q && (!q_out || n_heads < 1))) return fail(MTTS_E_INVALID, "append: missing arguments");
  if (S > KV_SLOTS_MAX) return fail(MTTS_E_INVALID, "append: at most 2^25 tokens a row");
  if (B * (int64_t)S > INT_MAX) return fail(MTTS_E_INVALID, "append: too many tokens");
  if (q && B * S > 1 && ldqo < (size_t)n_heads * c.D) return fail(MTTS_E_INVALID, "append: rows of q_out overlap");
  // (where its slots are is known on the device alone)
  const int64_t held = (int64_t)(mtts_kv_bytes(c.type, c.rows, c.n_kv, c.D, c.slots) / 2);
  for (const void* buf : {c.k, c.v})
    for (const auto& [src, ld] : {std::pair<const uint16_t*, size_t>(k, ldk), {v, ldv}})
      if (share(Runs(src, B * S, ld, 1, 0, (int64_t)c.n_kv * c.D), Runs(buf, 1, 0, 1, 0, held)))
        return fail(MTTS_E_INVALID, "append: k and v lie outside the cache");
  // (q may be rotated in place; the heads of other waves and the keys' and values' blocks may not be written)
  if (q) {
    const int M = B * S;
    const Runs o(q_out, M, ldqo, 1, 0, (int64_t)n_heads * c.D);
    if ((!(q == q_out && (M == 1 || ldq == ldqo)) && share(Runs(q, M, ldq, 1, 0, (int64_t)n_heads * c.D), o)) ||
        share(Runs(k, M, ldk, 1, 0, (int64_t)c.n_kv * c.D), o) || share(Runs(v, M, ldv, 1, 0, (int64_t)c.n_kv * c.D), o))
      return fail(MTTS_E_INVALID, "append: q_out overlaps q, k or v (q in place is fine, with its stride)");
  }
  KvAppendArgs a{c, q, k, v, ldq, ldk, ldv, q_out, ldqo, n_heads, qn, kn, eps, {}, pos, start, counts, B, S};
  if (!rope_of(rope, c.D, &a.r)) return fail(MTTS_E_INVALID, "append: rotary dim is even and at most the head's");
  HIPCHK(kv_append(a, (hipStream_t)stream));
  return 0;
}

extern "C" int mtts_k_kv_read(const mtts_kv_cache* cache, uint16_t* k_out, uint16_t* v_out, const int32_t* start,
                              const int32_t* counts, int B, int n, void* stream) {
  KV_CACHE(cache, c);
  if (B < 0 || B > c.rows || n < 0) return fail(MTTS_E_INVALID, "read: more rows than the cache has");
  if (B == 0 || n == 0) return 0;
  if (!k_out || !v_out || (((uintptr_t)k_out | (uintptr_t)v_out) & 15))
    return fail(MTTS_E_INVALID, "read: 16-byte aligned outputs");
  if (n > KV_SLOTS_MAX) return fail(MTTS_E_INVALID, "read: at most 2^25 slots");
  HIPCHK(kv_read(KvReadArgs{c, k_out, v_out, start, counts, B, n}, (hipStream_t)stream));
  return 0;
}

extern "C" int mtts_k_kv_compact(const mtts_kv_cache* cache, const int32_t* start, const int32_t* path,
                                 const int32_t* took, int B, int P, void* stream) {
  KV_CACHE(cache, c);
  if (B < 0 || B > c.rows || P < 0) return fail(MTTS_E_INVALID, "compact: more rows than the cache has");
  if (P > KV_PATH_MAX) return fail(MTTS_E_UNSUPPORTED, "compact: paths of at most 64 tokens");
  if (B == 0 || P == 0) return 0;
  if (!start || !path || !took) return fail(MTTS_E_INVALID, "compact: missing arguments");
  HIPCHK(kv_compact(KvCompactArgs{c, start, path, took, B, P}, (hipStream_t)stream));
  return 0;
}

extern "C" size_t mtts_k_attn_kv_ws_bytes(int B, int T, int n_heads, int n_kv, int D, int slots, int max_len) {
  if (B < 1 || T < 1 || n_kv < 1 || n_heads < n_kv || !dim_ok(D) || slots < 32) return 0;
  return attn_kv_ws_bytes(B, T, n_heads, n_kv, D, slots, max_len);
}

extern "C" int mtts_k_attn_kv(const mtts_kv_cache* cache, const uint16_t* q, size_t ldq, uint16_t* out, size_t ldo,
                              int n_heads, const int32_t* start, const int32_t* counts, const uint64_t* tree,
                              const uint8_t* mask, int B, int T, float scale, int max_len, void* ws, void* stream) {
  KV_CACHE(cache, c);
  if (B < 0 || B > c.rows || T < 0) return fail(MTTS_E_INVALID, "attention: more rows than the cache has");
  if (n_heads < 1 || n_heads % c.n_kv) return fail(MTTS_E_INVALID, "attention: q heads in groups of the KV heads");
  if (tree && T > KV_TREE_MAX) return fail(MTTS_E_UNSUPPORTED, "attention: trees of at most 64 tokens");
  if (B == 0 || T == 0) return 0;
  if (!q || !out || !start) return fail(MTTS_E_INVALID, "attention: missing arguments");
  if (((uintptr_t)q & 15) || ldq % 8 || ((uintptr_t)out & 7) || ldo % 4 || ((uintptr_t)mask & 7) || ((uintptr_t)tree & 7))
    return fail(MTTS_E_INVALID, "attention: q 16-byte and out 8-byte aligned, in every row; mask and tree 8-byte");
  if ((int64_t)B * T > 1 && ldo < (size_t)n_heads * c.D) return fail(MTTS_E_INVALID, "attention: rows of out overlap");
  if (B > 65535) return fail(MTTS_E_UNSUPPORTED, "attention: at most 65,535 rows");
  if ((int64_t)T * n_heads > (1 << 30) || (int64_t)B * T > INT_MAX) return fail(MTTS_E_INVALID, "attention: too many tokens");
  // (a block reads the q of the rows that it writes, before it writes them: in place is fine)
  if (!(q == out && (B * T == 1 || ldq == ldo)) &&
      share(Runs(q, B * T, ldq, 1, 0, (int64_t)n_heads * c.D), Runs(out, B * T, ldo, 1, 0, (int64_t)n_heads * c.D)))
    return fail(MTTS_E_INVALID, "attention: out overlaps q (in place is fine, with its stride)");
  if (!ws && attn_kv_ws_bytes(B, T, n_heads, c.n_kv, c.D, c.slots, max_len))
    return fail(MTTS_E_INVALID, "attention: workspace required");
  if ((uintptr_t)ws & 15) return fail(MTTS_E_INVALID, "attention: 16-byte aligned workspace");
  AttnKvArgs a{c, q, out, ldq, ldo, mask, start, counts, tree, (float*)ws, B, T, n_heads,
               scale > 0 ? scale : 1.0f / std::sqrt((float)c.D), max_len};
  HIPCHK(attn_kv(a, (hipStream_t)stream));
  return 0;
}
