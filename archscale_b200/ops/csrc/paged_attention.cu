// Entry of the attention over a paged key-value cache: which kernel takes a call, and its launches.
#include "paged_attention.cuh"

namespace b200 {

struct PaPlan { PaArgs p; int dt, nc, span, tiles, nrt, nb; bool gen, ok; };

static PaPlan pa_plan(const PagedView& c, const b200_paged_query& a) {
  PaPlan s = {};
  PaArgs& p = s.p;
  p.c = c; p.a = a;
  const int es = c.type == 2 ? 1 : 2, D = c.dim;
  p.page_b = c.k_page * es; p.group_b = c.k_group * es; p.slot_b = c.k_slot * es;
  const bool alike = c.k_page == c.v_page && c.k_group == c.v_group && c.k_slot == c.v_slot;
  const uint64_t where = reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v) | static_cast<uint64_t>(p.page_b | p.group_b | p.slot_b | D * es);
  p.piece = where % 16 == 0 ? 16 : where % 8 == 0 ? 8 : where % 4 == 0 ? 4 : 0;
  s.ok = a.type == 1 && c.type != 0 && alike && p.piece != 0 && D <= (a.diff ? 128 : 256);
  if (!s.ok) return s;
  p.per = a.H / c.groups;                                                       // query heads, or pairs of them, of a key head or pair
  const int64_t rows = static_cast<int64_t>(p.per) * a.T;
  s.ok = rows <= 0x7fff0000LL;                                                  // counted in 32 bits, tiles of them rounded up
  if (!s.ok) return s;
  p.rows = static_cast<int>(rows);
  p.heads = a.diff ? c.groups / 2 : c.groups;
  s.nc = p.rows <= (a.diff ? 4 : 8) ? 1 : 2;
  s.dt = a.diff ? (D <= 64 ? 128 : 256) : D <= 64 ? 64 : D <= 128 ? 128 : 256;
  const int64_t far = (static_cast<int64_t>(c.pages) * p.page_b + static_cast<int64_t>(c.page_size) * p.slot_b) / 16;
  p.page_16 = static_cast<uint32_t>(p.page_b / 16); p.slot_16 = static_cast<uint32_t>(p.slot_b / 16);
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i) if (c.page_size == 1 << i) p.page_shift = i;
  const int64_t far_s = static_cast<int64_t>(c.pages) * (c.ks_page > c.vs_page ? c.ks_page : c.vs_page) + static_cast<int64_t>(c.page_size) * (c.ks_slot > c.vs_slot ? c.ks_slot : c.vs_slot);
  p.ks_page = static_cast<uint32_t>(c.ks_page); p.ks_slot = static_cast<uint32_t>(c.ks_slot);
  p.vs_page = static_cast<uint32_t>(c.vs_page); p.vs_slot = static_cast<uint32_t>(c.vs_slot);
  s.gen = far > 0xffffffffLL || far_s > 0xffffffffLL || p.piece != 16 || D != (a.diff ? s.dt / 2 : s.dt);
  p.same_scales = p.ks_page == p.vs_page && p.ks_slot == p.vs_slot;
  p.q_wide = reinterpret_cast<uintptr_t>(a.q) % 8 == 0 && (a.q_batch | a.q_token | a.q_head) % 4 == 0;
  p.q_words = reinterpret_cast<uintptr_t>(a.q) % 4 == 0 && (a.q_batch | a.q_token | a.q_head) % 2 == 0;
  const int qrows = (a.diff ? 4 : 8) * s.nc;
  const int64_t room = static_cast<int64_t>(c.table_cols) * c.page_size, seen = a.window >= 0 ? static_cast<int64_t>(a.window) + qrows + 1 : room;
  const int64_t span = room < seen ? room : seen;
  s.span = static_cast<int>(span < 0x7fffff00 ? span : 0x7fffff00);
  s.tiles = (p.rows + qrows - 1) / qrows;
  s.nrt = s.tiles < PA_ENTRIES ? s.tiles : PA_ENTRIES;
  s.nb = PA_ENTRIES / s.nrt;
  const int64_t fit = 0x40000000LL / (static_cast<int64_t>(s.nrt) * p.heads * (s.span / 64 + 1));       // chunks are counted in 32 bits
  if (fit < 1) { s.ok = false; return s; }
  if (s.nb > fit) s.nb = static_cast<int>(fit);
  if (s.nb > a.B) s.nb = a.B;
  return s;
}
static int pa_go(const PaPlan& s, PaArgs& p, int num_sms, void* ws, int64_t* need, cudaStream_t st) {
  return (p.c.type == 2 ? pa_run_e4m3 : pa_run_bf16)(p, s.dt, p.a.diff != 0, s.nc, s.gen, s.span, num_sms, ws, need, st);
}

}  // namespace b200

extern "C" int64_t b200_paged_attention_workspace(const b200_paged_view* c, const b200_paged_query* a, int num_sms) {
  using namespace b200;
  if (a->B <= 0 || a->T <= 0 || a->H <= 0) return 0;
  PaPlan s = pa_plan(*c, *a);
  if (!s.ok) return 0;
  s.p.nb = s.nb; s.p.nrt = s.nrt;
  int64_t need = 0;
  pa_go(s, s.p, num_sms, nullptr, &need, nullptr);
  return need;
}

extern "C" int b200_paged_attention(const b200_paged_view* c, const b200_paged_query* a, void* ws, int num_sms, cudaStream_t st) {
  using namespace b200;
  if (a->B <= 0 || a->T <= 0 || a->H <= 0) return 0;
  PaPlan s = pa_plan(*c, *a);
  if (!s.ok) return b200_paged_attention_rows(c, a, st);
  for (int b = 0; b < a->B; b += s.nb)
    for (int rt = 0; rt < s.tiles; rt += s.nrt) {
      s.p.b0 = b; s.p.nb = a->B - b < s.nb ? a->B - b : s.nb;
      s.p.rt0 = rt; s.p.nrt = s.tiles - rt < s.nrt ? s.tiles - rt : s.nrt;
      if (const int rc = pa_go(s, s.p, num_sms, ws, nullptr, st)) return rc;
    }
  return 0;
}
