// The sums by bucket of the dense-band layers: against sums on the host, and with a tile that says that one of its waits ran out.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include "gk_terms_band.cuh"

using namespace gk;
using namespace gk::banded;

#define OK(call)                                                       \
  do {                                                                 \
    const int rc_ = (int)(call);                                       \
    if (rc_) { printf("line %d: %s -> %d\n", __LINE__, #call, rc_); return 1; } \
  } while (0)

static unsigned next(unsigned& s) { return s = s * 1664525u + 1013904223u; }

static int sums(int tiles, int pitch, int H, int maps, int buckets) {
  const int columns = H * maps;
  BandRoom r;
  r.elements = (long long)tiles * pitch * kTileM;
  r.sum = band_sum_shape(r.elements, buckets, columns);
  const size_t n = (size_t)r.elements, cells = (size_t)buckets * columns;
  std::vector<unsigned char> ids(n), low(n * columns);
  std::vector<unsigned short> up(n * columns);
  std::vector<double> want(cells), size(cells);
  std::vector<float> got(cells), first(cells);
  std::vector<int> dirty((size_t)H * tiles);
  unsigned seed = 7;
  for (auto& i : ids) { const unsigned x = next(seed) >> 16; i = x % 5 ? x % buckets : 255; }
  for (size_t i = 0; i < n * columns; ++i) {
    const bool part = ids[i % n] != 255;
    float g = part ? (float)((int)(next(seed) >> 8) - (1 << 23)) * 1e-6f : 0.f;
    unsigned bits;
    memcpy(&bits, &g, 4);
    up[i] = (unsigned short)(bits >> 16);
    low[i] = (unsigned char)(bits >> 8);
    bits &= ~255u;
    memcpy(&g, &bits, 4);
    if (part) {
      want[(size_t)ids[i % n] * columns + i / n] += g;
      size[(size_t)ids[i % n] * columns + i / n] += std::fabs(g);
    }
  }
  float* out;
  OK(cudaMalloc(&r.ids, n));
  OK(cudaMalloc(&r.g, n * columns * 2));
  OK(cudaMalloc(&r.g_low, n * columns));
  OK(cudaMalloc(&r.dirty, dirty.size() * sizeof(int)));
  OK(cudaMalloc(&r.partial, r.sum.blocks * cells * sizeof(double)));
  OK(cudaMalloc(&out, cells * sizeof(float)));
  OK(cudaMemcpy(r.ids, ids.data(), n, cudaMemcpyHostToDevice));
  OK(cudaMemcpy(r.g, up.data(), n * columns * 2, cudaMemcpyHostToDevice));
  OK(cudaMemcpy(r.g_low, low.data(), n * columns, cudaMemcpyHostToDevice));
  const int head = H - 1;
  for (int lost : {-1, 0, tiles - 1}) {
    for (auto& d : dirty) d = 0;
    dirty[0] = kTileAgain;                          // done again: its sums are known
    if (lost >= 0) dirty[(size_t)head * tiles + lost] = kTileLost;
    OK(cudaMemcpy(r.dirty, dirty.data(), dirty.size() * sizeof(int), cudaMemcpyHostToDevice));
    OK(run_band_bucket_sum(r, tiles, buckets, H, maps, out, (cudaStream_t)0));
    OK(cudaMemcpy(got.data(), out, cells * sizeof(float), cudaMemcpyDeviceToHost));
    for (size_t i = 0; i < cells; ++i) {
      const bool gone = lost >= 0 && (int)(i % columns) / maps == head;
      // float32 sums in any order: n roundings of 2^-24 of the magnitudes at the most
      const double bound = size[i] * 6e-8 * (2.0 + (double)n / buckets) + 1e-30;
      if (gone ? !std::isnan(got[i]) : !(std::fabs(got[i] - want[i]) <= bound) || (lost >= 0 && got[i] != first[i])) {
        printf("%d tiles, %d buckets, lost %d: cell %zu is %g, not %g\n", tiles, buckets, lost, i, got[i], gone ? NAN : want[i]);
        return 1;
      }
    }
    if (lost < 0) first = got;
  }
  for (void* p : {(void*)r.ids, (void*)r.g, (void*)r.g_low, (void*)r.dirty, (void*)r.partial, (void*)out}) OK(cudaFree(p));
  return 0;
}

int main() {
  for (const auto& z : {std::vector<int>{1, 64, 1, 1, 7}, {3, 128, 2, 2, 32}, {300, 64, 3, 1, 100}, {5, 384, 2, 2, 255}})
    if (sums(z[0], z[1], z[2], z[3], z[4])) return 1;
  printf("fine\n");
  return 0;
}
