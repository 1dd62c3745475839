// Host only: for every shape of the layers with learned score terms, the bytes that a call takes of its workspace, in the order in which
// gk_terms.cuh takes them and in the geometries that its launches pick, against what terms_bytes asks the caller for.
#include <cstdio>

#include "gk_terms.cuh"

using namespace gk;

namespace {
long long checked = 0, short_by = 0;
char worst[256] = "";

template <template <class> class Op, typename T>
void take_walk(Arena& ar, const GeoPick& s, long long tiles) {
  dispatch_geo<T, false, true>(s, [&](auto tag) -> int {
    using O = Op<typename decltype(tag)::type>;
    const size_t slots = (size_t)s.nhb * 2 * tiles;
    ar.take(slots * O::kCarryElems * sizeof(typename O::A));
    ar.take(slots * 4);
    return 0;
  });
}
template <class G> using Fwd1 = TermsFwd<G, 1, true>;
template <class G> using Fwd2 = TermsFwd<G, 2, true>;
template <class G> using Dst1 = TermsBwdDst<G, 1, true>;
template <class G> using Dst2 = TermsBwdDst<G, 2, true>;

void take_graph(Arena& ar, long long E, long long n, int index_bytes, bool eid) {
  ar.take(sizeof(PlanHeader));
  ar.take((size_t)E * 4);
  ar.take((size_t)(tile_count(E, n, tile_cost(E, n)) + 1) * 4);
  if (index_bytes == 8) ar.take((size_t)E * 4);
  if (index_bytes == 8 && eid) ar.take((size_t)E * 4);
}

template <typename T>
void shapes(long long E, long long n_dst, long long n_src, int index_bytes) {
  using A = typename AccOf<T>::type;
  const long long n = n_dst > n_src ? n_dst : n_src, tiles = tile_count(E, n_dst, tile_cost(E, n_dst)),
                  tiles_t = tile_count(E, n_src, tile_cost(E, n_src));
  for (int diff = 0; diff < 2; ++diff)
    for (int buckets : {0, 32, 16384})
      for (int D = 1; D <= 2048; ++D)
        for (int H = 1; H <= 256; ++H) {
          if (!diff && !buckets) continue;
          TermsCall<T> c{};
          c.diff = diff; c.H = H; c.D = D; c.buckets = buckets; c.E = E; c.n_dst = n_dst; c.n_src = n_src;
          GeoPick s;
          if (terms_check(c, 1, true, &s) != GRAPHOP_OK) continue;
          const int columns = H * c.maps();
          const auto report = [&](const char* what, const Arena& ar, bool backward) {
            const size_t asked = terms_bytes(diff, backward, E, n, H, D, buckets, sizeof(T), index_bytes);
            ++checked;
            if (ar.used > asked && (long long)(ar.used - asked) > short_by) {
              short_by = (long long)(ar.used - asked);
              snprintf(worst, sizeof worst, "%s, %d-byte elements, %d maps, H %d, D %d, %d buckets, %lld edges, %lld and %lld nodes", what,
                       (int)sizeof(T), c.maps(), H, D, buckets, E, n_dst, n_src);
            }
          };
          {
            Arena ar(nullptr, 0);
            take_graph(ar, E, n_dst, index_bytes, false);
            if (diff) take_walk<Fwd2, T>(ar, s, tiles);
            else take_walk<Fwd1, T>(ar, s, tiles);
            report("forward", ar, false);
          }
          Arena ar(nullptr, 0);
          ar.take((size_t)E * stat_heads(columns, (int)sizeof(A)) * sizeof(EdgePair<A>));
          if (diff) ar.take((size_t)n_dst * H * sizeof(A));
          const size_t mark = ar.used;
          take_graph(ar, E, n_dst, index_bytes, false);
          if (diff) take_walk<Dst2, T>(ar, s, tiles);
          else take_walk<Dst1, T>(ar, s, tiles);
          if (buckets) ar.take((size_t)bucket_shape(E, columns, buckets, (int)sizeof(A)).blocks * buckets * columns * sizeof(double));
          if (diff) ar.take((size_t)bucket_shape(n_dst, H, 1, (int)sizeof(A)).blocks * H * sizeof(double));
          report("destination side", ar, true);
          ar.used = mark;
          take_graph(ar, E, n_src, index_bytes, true);
          const size_t before = ar.used;
          take_walk<TermsBwdSrc, T>(ar, terms_geo(columns, D, sizeof(T)), tiles_t);
          report("source side", ar, true);
          if constexpr (kSumsByRegister<T>) {
            ar.used = before;
            const GeoPick p = pick_sum_geo(columns, D, sizeof(T), 16);
            dispatch_sum_geo<T, false>(p, [&](auto tag) -> int {
              using O = TermsSumPairs<typename decltype(tag)::type>;
              const size_t slots = (size_t)p.nhb * 2 * tiles_t;
              ar.take(slots * O::kCarryElems * sizeof(A));
              ar.take(slots * 4);
              return 0;
            });
            report("source side by the summing walker", ar, true);
          }
        }
}
}  // namespace

int main() {
  const long long sizes[][3] = {{1, 1, 1}, {1000, 10, 3000}, {300000, 100000, 100000}, {4000000, 200000, 1000}, {90000000, 3000000, 5000000}};
  for (const auto& z : sizes)
    for (int index_bytes : {4, 8}) {
      shapes<float>(z[0], z[1], z[2], index_bytes);
      shapes<double>(z[0], z[1], z[2], index_bytes);
      shapes<__nv_bfloat16>(z[0], z[1], z[2], index_bytes);
    }
  if (short_by) {
    printf("short by %lld bytes: %s\n", short_by, worst);
    return 1;
  }
  printf("%lld calls fit\n", checked);
  return checked < 10000;
}
