// The rules of immerdink_b200/csrc/linear/choice.hpp for a host test: nothing is launched or dereferenced.
#include "linear/choice.hpp"

namespace {
const void* at(int64_t p) { return reinterpret_cast<const void*>(p); }
imd::LinearArgs args(imd::WeightKind kind, int64_t rows, int64_t n, int64_t k, int64_t x, int64_t xs, int64_t w, int64_t ws, int group) {
  imd::LinearArgs a{};
  a.kind = kind, a.rows = rows, a.n = n, a.k = k, a.x = at(x), a.x_stride = xs, a.w = at(w), a.w_stride = ws, a.group = group;
  return a;
}
}  // namespace

extern "C" {
// 's' streamed, 't' tensor cores with x by TMA, 'a' tensor cores with x brought by loads, 'm' the small kernel
int choice_w4(int64_t rows, int64_t n, int64_t k, int64_t x, int64_t xs, int64_t w, int64_t ws, int group) {
  const imd::LinearArgs a = args(imd::WeightKind::kU4, rows, n, k, x, xs, w, ws, group);
  const int clusters[4] = {148, 74, 33, 15};
  if (imd::stream_takes(a, clusters)) return 's';
  return !imd::dense4_takes(a) ? 'm' : imd::x4_for_tma(a) ? 't' : 'a';
}
int choice_8(int e4m3, int64_t rows, int64_t n, int64_t k, int64_t x, int64_t xs, int64_t w, int64_t ws) {
  const imd::LinearArgs a = args(e4m3 ? imd::WeightKind::kE4M3 : imd::WeightKind::kI8, rows, n, k, x, xs, w, ws, 0);
  return !imd::dense8_takes(a) ? 'm' : imd::both8_for_tma(a) ? 't' : 'a';
}
int w4_by_tma(int64_t n, int64_t k, int64_t w, int64_t ws) {
  return imd::w4_for_tma(args(imd::WeightKind::kU4, 1, n, k, 0, 0, w, ws, 128));
}
int split(int64_t tiles, int64_t steps, int c1, int c2, int c4, int c8, int per_sm) {
  const int clusters[4] = {c1, c2, c4, c8};
  return imd::split_of(tiles, steps, clusters, per_sm);
}
}
