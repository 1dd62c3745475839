// Attention with learned score terms: a bias by buckets, and differential attention.
//
// With n a node, j a position of its CSR row, c = other[j], s the scale:
//     bucket   S[j, h] = s q[n, h].k[c, h] + T[b[j], h];     p = softmax of S over n's positions;     o[n, h] = sum_j p[j, h] v[c, h]
//     diff     p1, p2 the same of the maps 2h and 2h + 1 of q and k (with T or without);     o[n, h] = sum_j (p1 - lam[h] p2) v[c, h]
// A position takes no part where its bucket is no row of the table or where the table's entry is at most kMaskedBias (-inf, the
// lowest values of a type): its rows are not multiplied with anything, so that NaN there stays there.  A node of which nothing
// takes part is one without edges: o = 0, lse = -inf, no gradients.
//
// Backward, with dp = dO.v and t = dO.o (of either map's own sum, o1 and o2):
//     g1 = p1 (dp - t1), g2 = -lam p2 (dp - t2);     dq = s sum g k;  dk = s sum g q;  dv = sum (p1 - lam p2) dO;
//     dT[b, h] = sum of g over the positions of bucket b;     dlam = - sum of t2 over the nodes
// The destination side leaves (p1 - lam p2, g) of every position and map; the source side and dT are sums of them.
//
// All are walks of gk_group.cuh, bound like the plain layer by the gathered rows.  A pair of maps of d features is one head of
// D = 2 d features of v: the row of the node's pair of q, of k, of v and of o lie at the same offsets, so that one geometry
// serves all of them, and both maps are formed in one walk that gathers v once.
#pragma once
#include "gk_host.cuh"

namespace gk {

constexpr double kMaskedBias = -1e38;

// The scores of both kernels, in base-2 units.  Lanes of one slot (W == 1): the lower half of a head's lanes holds map 0, the
// upper half map 1; with more slots the lower half of the slots does.  Either way every lane ends with the scores of all maps.
template <class GEO, int kMaps>
struct TermsScores {
  using A = typename GEO::A;
  using F = typename GEO::F;
  static constexpr int W = GEO::W, V = GEO::V;
  static constexpr bool kHalves = kMaps == 2 && W == 1;   // a lane's slot belongs to one map
  static __device__ __forceinline__ bool upper(const GEO& geo) { return (threadIdx.x & (geo.lanes_per_head() >> 1)) != 0; }
  static __device__ __forceinline__ void partial(A (&s)[kMaps], const F (&q)[W], const F (&k)[W]) {
    if constexpr (kMaps == 1 || kHalves) {
      s[0] = frag_dot<V, W>(q, k);
    } else {
      constexpr int N = W / 2;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        F x[N], y[N];
#pragma unroll
        for (int i = 0; i < N; ++i) { x[i] = q[m * N + i]; y[i] = k[m * N + i]; }
        s[m] = frag_dot<V, N>(x, y);
      }
    }
  }
  static __device__ __forceinline__ void finish(const GEO& geo, A (&s)[kMaps]) {
    if constexpr (kHalves) {
      const int half = geo.lanes_per_head() >> 1;
      A own = s[0];
      if constexpr (GEO::LT > 0) {
#pragma unroll
        for (int o = 1; o < GEO::LT / 2; o <<= 1) own += __shfl_xor_sync(kFull, own, o);
      } else {
        for (int o = 1; o < half; o <<= 1) own += __shfl_xor_sync(kFull, own, o);
      }
      const A oth = __shfl_xor_sync(kFull, own, half);
      const bool up = upper(geo);
      s[0] = up ? oth : own;
      s[1] = up ? own : oth;
    } else {
#pragma unroll
      for (int m = 0; m < kMaps; ++m) s[m] = geo.head_sum(s[m]);
    }
  }
  // the map that slot i of this lane belongs to
  static __device__ __forceinline__ A of_slot(const A (&x)[kMaps], int i, bool up) {
    if constexpr (kMaps == 1) return x[0];
    else if constexpr (kHalves) return up ? x[1] : x[0];
    else return x[i >= W / 2];
  }
};

// The bias of a position's maps, as it waits in the walker's table: in base-2 units, -inf where the position takes no part.
template <class GEO, int kMaps>
struct TermsBias {
  using T = typename GEO::T;
  using A = typename GEO::A;
  struct Raw { T t[kMaps]; };
  static constexpr int kBytes = kMaps * (int)sizeof(A);
  static __device__ __forceinline__ Raw fetch(const T* table, int maps, int head, int bucket, bool live) {
    Raw r;
#pragma unroll
    for (int m = 0; m < kMaps; ++m)
      r.t[m] = live ? __ldg(table + ((long long)bucket * maps + head * kMaps + m)) : from_acc<T>(neg_inf<A>());
    return r;
  }
  static __device__ __forceinline__ void put(unsigned at, const Raw& r) {
    A x[kMaps];
#pragma unroll
    for (int m = 0; m < kMaps; ++m) {
      const A b = to_acc<T>(r.t[m]);
      x[m] = b <= A(kMaskedBias) ? neg_inf<A>() : b * A(kLog2e);
    }
#pragma unroll
    for (int m = 0; m < kMaps; ++m) {
      if constexpr (sizeof(A) == 4) asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + m * 4), "f"(x[m]) : "memory");
      else asm volatile("st.shared.f64 [%0], %1;" ::"r"(at + m * 8), "d"(x[m]) : "memory");
    }
  }
  static __device__ __forceinline__ void get(A (&b)[kMaps], unsigned at) {
    if constexpr (kMaps == 1) lds(b[0], at);
    else lds2(b[0], b[1], at);
  }
};

// Two maps of 2-byte elements: registers that the maps and the table's addresses take beyond the fragments, in fragments.  R-MAT 16, 8
// pairs of 64 with a bias, forward 1217 us with none more (108 bytes a thread spill), 1018 with one, 1102 with four (nothing spills, 16
// warps per SM); 600 thousand edges, 3 pairs of 32, destination side 226 us with none more, 188 with three.
template <class GEO, int kMaps, bool kBucket>
constexpr int kTermsMoreFwd = kMaps == 2 && sizeof(typename GEO::T) == 2 ? 1 : 0;
template <class GEO, int kMaps, bool kBucket>
constexpr int kTermsMoreDst = kMaps == 2 && kBucket && sizeof(typename GEO::T) == 2 ? 3 : 0;

template <class GEO, int kMaps, bool kBucket>
struct TermsFwd : GEO, Shape<GEO, 2, kBucket ? TermsBias<GEO, kMaps>::kBytes : 0, 1 + kMaps + kTermsMoreFwd<GEO, kMaps, kBucket>, 1, 0, 2,
                         (sizeof(typename GEO::T) > 2)> {
  using T = typename GEO::T;
  using A = typename GEO::A;
  using F = typename GEO::F;
  using Scores = TermsScores<GEO, kMaps>;
  using Bias = TermsBias<GEO, kMaps>;
  using Raw = typename Bias::Raw;
  static constexpr int W = GEO::W, V = GEO::V, kRow = GEO::kRow;   // rows of a ring step: k, v
  static constexpr const char* kName = kMaps == 2 ? "attention_diff_fwd" : "attention_bucket_fwd";
  static constexpr bool kRowOut = true, kUsesOther = true, kUsesEid = kBucket, kFoldsEid = false, kComputed = kBucket, kMasks = kBucket;
  const T* __restrict__ q;
  const T* __restrict__ k;
  const T* __restrict__ v;
  const T* __restrict__ table;   // (buckets, H * kMaps)
  const T* __restrict__ lam;     // (H)
  T* __restrict__ o;
  A* __restrict__ each;          // (n, H, kMaps, D): every map's own sum as it is, for the backward; may be null
  A* __restrict__ lse;           // (n, H * kMaps)
  A scale;
  int buckets;
  struct State {
    typename GEO::Lane ln;
    const unsigned char *kb, *vb;
    F q[W], acc[kMaps][W];
    A m[kMaps], l[kMaps];
  };
  struct Carry { F x[kMaps][W]; A m[kMaps], l[kMaps]; };
  __device__ __forceinline__ void setup(State& st, int gl, int hb) const {
    st.ln = this->lane_of(gl, hb);
    st.kb = reinterpret_cast<const unsigned char*>(k + st.ln.off);
    st.vb = reinterpret_cast<const unsigned char*>(v + st.ln.off);
    begin_merge(st);
#pragma unroll
    for (int i = 0; i < W; ++i) st.q[i].zero();
  }
  __device__ __forceinline__ bool takes_part(int b) const { return (unsigned)b < (unsigned)buckets; }
  __device__ __forceinline__ Raw raw_scalar(int h, int b, bool live) const { return Bias::fetch(table, this->H * kMaps, h, b, live); }
  __device__ __forceinline__ void put_scalar(unsigned at, const Raw& r) const { Bias::put(at, r); }
  __device__ __forceinline__ const void* scalar_of(int, int, int) const { return nullptr; }
  __device__ __forceinline__ void stage(const State& st, unsigned slot, int id, int, bool live) const {
    this->stage_row(st.ln, slot, st.kb, id, this->rowb, live);
    this->stage_row(st.ln, slot + kRow, st.vb, id, this->rowb, live);
  }
  template <int N>
  __device__ __forceinline__ void fold(State& st, unsigned slot, unsigned tab, const bool (&active)[N], unsigned,
                                       const int (&)[N]) const {
    A s[N][kMaps], mn[kMaps], ref[kMaps];
#pragma unroll
    for (int v = 0; v < N; ++v) {
      F f[W];
      this->load_staged(f, slot + v * this->kStepBytes);
      Scores::partial(s[v], st.q, f);
    }
#pragma unroll
    for (int m = 0; m < kMaps; ++m) mn[m] = st.m[m];
#pragma unroll
    for (int v = 0; v < N; ++v) {
      Scores::finish(*this, s[v]);
      if constexpr (kBucket) {
        A b[kMaps];
        Bias::get(b, tab + v * GEO::kHeads * Bias::kBytes);
#pragma unroll
        for (int m = 0; m < kMaps; ++m) s[v][m] = b[m] == neg_inf<A>() ? b[m] : s[v][m] + b[m];
      }
#pragma unroll
      for (int m = 0; m < kMaps; ++m) {
        if (!kBucket && !active[v]) s[v][m] = neg_inf<A>();
        mn[m] = s[v][m] > mn[m] ? s[v][m] : mn[m];
      }
    }
    // The sums are relative to a reference that may lag behind the maximum by up to 2^8 (the rounding is relative), so that after a
    // node's first edges they are seldom rescaled.
    bool grows = false;
#pragma unroll
    for (int m = 0; m < kMaps; ++m) grows = grows || mn[m] > st.m[m] + A(8);   // m = -inf before a node's first edge
    if (__any_sync(kFull, grows)) {
#pragma unroll
      for (int m = 0; m < kMaps; ++m) {
        const A corr = st.m[m] == mn[m] ? A(1) : gk_exp2(st.m[m] - mn[m]);
        st.m[m] = mn[m];
        st.l[m] *= corr;
#pragma unroll
        for (int i = 0; i < W; ++i) st.acc[m][i].scale(corr);
      }
    }
#pragma unroll
    for (int m = 0; m < kMaps; ++m) ref[m] = st.m[m] == neg_inf<A>() ? A(0) : st.m[m];   // nothing has taken part so far: 2^-inf
#pragma unroll
    for (int v = 0; v < N; ++v) {
      F f[W];
      this->load_staged(f, slot + v * this->kStepBytes + kRow);
#pragma unroll
      for (int m = 0; m < kMaps; ++m) {
        const A p = gk_exp2(s[v][m] - ref[m]);
        st.l[m] += p;
        if (!kBucket || p != A(0)) {   // a masked row may hold anything
#pragma unroll
          for (int i = 0; i < W; ++i) st.acc[m][i].axpy(p, f[i]);
        }
      }
    }
  }
  __device__ __forceinline__ void stage_node(const State& st, unsigned buf, int, int node) const {
    this->stage_row(st.ln, buf, reinterpret_cast<const unsigned char*>(q + st.ln.off), node, this->rowb, true);
  }
  __device__ __forceinline__ void begin(State& st, unsigned buf, int) const {
    this->load_staged(st.q, buf);
    begin_merge(st);
    const A c = scale * A(kLog2e);
#pragma unroll
    for (int i = 0; i < W; ++i) st.q[i].scale(c);
  }
  __device__ __forceinline__ void began(State&, int, bool) const {}
  // o is rounded to the element type, and dO . o out of it would carry that into every score gradient (two-byte elements, 5 edges a
  // node: dq 2.6e-3 off float64 instead of 1.7e-3): the backward gets the sums unrounded
  __device__ __forceinline__ void store_sums(const State& st, long long node, int m, const F (&x)[W]) const {
    A* at = each + (kMaps * node * this->HD + (long long)(kMaps - 1) * st.ln.head * this->D + (long long)m * this->D + st.ln.off);
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (this->has(st.ln, i)) frag_save<A, V>(at + i * this->slot_step(), x[i]);
  }
  __device__ __forceinline__ void store_row(const State& st, int node) const {
    F out[W];
#pragma unroll
    for (int m = 0; m < kMaps; ++m) {
      const A inv = st.l[m] == A(0) ? A(0) : A(1) / st.l[m];
      F x[W];
#pragma unroll
      for (int i = 0; i < W; ++i) { x[i] = st.acc[m][i]; x[i].scale(inv); }
      if (each) store_sums(st, node, m, x);
      const A c = m == 0 ? A(1) : -to_acc<T>(__ldg(lam + st.ln.head));
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if (m == 0) out[i] = x[i];
        else out[i].axpy(c, x[i]);
      }
      // m is a base-2 exponent: lse = (m + log2 l) * ln 2, -inf where nothing took part
      if (st.ln.first)
        lse[((long long)node * this->H + st.ln.head) * kMaps + m] = (st.m[m] + gk_log2(st.l[m])) * A(kLn2);
    }
    this->store_row_slots(st.ln, o + (long long)node * this->HD + st.ln.off, out);
  }
  __device__ __forceinline__ void zero_row(const State& st, long long n) const {
    this->zero_slots(st.ln, o, n);
    F z[W];
#pragma unroll
    for (int i = 0; i < W; ++i) z[i].zero();
#pragma unroll
    for (int m = 0; m < kMaps; ++m) {
      if (each) store_sums(st, n, m, z);
      if (st.ln.first) lse[(n * this->H + st.ln.head) * kMaps + m] = neg_inf<A>();
    }
  }
  static constexpr int kCarryElems = kMaps * (GEO::kAccs + 2 * GEO::G);
  __device__ __forceinline__ void begin_merge(State& st) const {
#pragma unroll
    for (int m = 0; m < kMaps; ++m) {
      st.m[m] = neg_inf<A>();
      st.l[m] = A(0);
#pragma unroll
      for (int i = 0; i < W; ++i) st.acc[m][i].zero();
    }
  }
  __device__ __forceinline__ void save_carry(const State& st, A* rec, int gl) const {
#pragma unroll
    for (int m = 0; m < kMaps; ++m) {
      this->save_acc(rec + m * GEO::kAccs, gl, st.acc[m]);
      rec[kMaps * GEO::kAccs + 2 * m * GEO::G + gl] = st.m[m];
      rec[kMaps * GEO::kAccs + (2 * m + 1) * GEO::G + gl] = st.l[m];
    }
  }
  __device__ __forceinline__ void load_carry(Carry& c, const A* rec, int gl) const {
#pragma unroll
    for (int m = 0; m < kMaps; ++m) {
      this->load_acc_raw(c.x[m], rec + m * GEO::kAccs, gl);
      c.m[m] = rec[kMaps * GEO::kAccs + 2 * m * GEO::G + gl];
      c.l[m] = rec[kMaps * GEO::kAccs + (2 * m + 1) * GEO::G + gl];
    }
  }
  __device__ __forceinline__ void merge(State& st, const Carry& c) const {
#pragma unroll
    for (int m = 0; m < kMaps; ++m) {
      const A mn = c.m[m] > st.m[m] ? c.m[m] : st.m[m];
      // a neutral partial has m = -inf: its weight is zero, never 2^(-inf - -inf)
      const A wa = st.m[m] == neg_inf<A>() ? A(0) : gk_exp2(st.m[m] - mn);
      const A wb = c.m[m] == neg_inf<A>() ? A(0) : gk_exp2(c.m[m] - mn);
      st.l[m] = st.l[m] * wa + c.l[m] * wb;
#pragma unroll
      for (int i = 0; i < W; ++i) st.acc[m][i].blend(wa, c.x[m][i], wb);
      st.m[m] = mn;
    }
  }
};

// Destination side of the backward: dq, the pairs (p1 - lam p2, g) per position and map, t2 per node for dlam.
template <class GEO, int kMaps, bool kBucket>
struct TermsBwdDst : GEO, Shape<GEO, 2, kBucket ? TermsBias<GEO, kMaps>::kBytes : 0, 4 + kTermsMoreDst<GEO, kMaps, kBucket>,
                            2 + kMaps * (int)(sizeof(typename GEO::A) / sizeof(typename GEO::T)), kMaps * (int)sizeof(typename GEO::A),
                            (sizeof(typename GEO::T) == 2 ? 2 : 1), true> {
  using T = typename GEO::T;
  using A = typename GEO::A;
  using F = typename GEO::F;
  using Scores = TermsScores<GEO, kMaps>;
  using Bias = TermsBias<GEO, kMaps>;
  using Raw = typename Bias::Raw;
  static constexpr int W = GEO::W, V = GEO::V, kRow = GEO::kRow;   // rows of a ring step: k, v; of a node: q, dO, the sum of every map
  static constexpr int kPer = (int)(sizeof(A) / sizeof(T));        // rows that a sum's row of wider elements fills
  static constexpr const char* kName = kMaps == 2 ? "attention_diff_bwd_dst" : "attention_bucket_bwd_dst";
  static constexpr bool kRowOut = true, kUsesOther = true, kUsesEid = kBucket, kFoldsEid = false, kComputed = kBucket, kMasks = kBucket;
  const T* __restrict__ q;
  const T* __restrict__ k;
  const T* __restrict__ v;
  const T* __restrict__ table;
  const T* __restrict__ lam;
  const A* __restrict__ sums;      // (n, H, kMaps, D), unrounded
  const T* __restrict__ dout;
  const A* __restrict__ lse;
  EdgePair<A>* __restrict__ pd;    // (E, Hp)
  A* __restrict__ t2;              // (n, H), kMaps == 2
  T* __restrict__ dq;
  A scale;
  int Hp, buckets;
  struct State {
    typename GEO::Lane ln;
    const unsigned char *kb, *vb;
    F q[W], gr[W], acc[W];
    A lse2[kMaps], delta[kMaps], lam;
  };
  struct Carry { F x[W]; };
  __device__ __forceinline__ void setup(State& st, int gl, int hb) const {
    st.ln = this->lane_of(gl, hb);
    st.kb = reinterpret_cast<const unsigned char*>(k + st.ln.off);
    st.vb = reinterpret_cast<const unsigned char*>(v + st.ln.off);
    begin_merge(st);
    st.lam = kMaps == 2 ? to_acc<T>(__ldg(lam + st.ln.head)) : A(0);
#pragma unroll
    for (int m = 0; m < kMaps; ++m) st.lse2[m] = st.delta[m] = A(0);
#pragma unroll
    for (int i = 0; i < W; ++i) { st.q[i].zero(); st.gr[i].zero(); }
  }
  __device__ __forceinline__ bool takes_part(int b) const { return (unsigned)b < (unsigned)buckets; }
  __device__ __forceinline__ Raw raw_scalar(int h, int b, bool live) const { return Bias::fetch(table, this->H * kMaps, h, b, live); }
  __device__ __forceinline__ void put_scalar(unsigned at, const Raw& r) const { Bias::put(at, r); }
  __device__ __forceinline__ const void* scalar_of(int, int, int) const { return nullptr; }
  __device__ __forceinline__ void stage(const State& st, unsigned slot, int id, int, bool live) const {
    this->stage_row(st.ln, slot, st.kb, id, this->rowb, live);
    this->stage_row(st.ln, slot + kRow, st.vb, id, this->rowb, live);
  }
  template <int N>
  __device__ __forceinline__ void fold(State& st, unsigned slot, unsigned tab, const bool (&active)[N], unsigned pos,
                                       const int (&)[N]) const {
    A s[N][kMaps], dp[N];
    F f[N][W];
#pragma unroll
    for (int v = 0; v < N; ++v) {
      this->load_staged(f[v], slot + v * this->kStepBytes + kRow);
      dp[v] = frag_dot<V, W>(st.gr, f[v]);
      this->load_staged(f[v], slot + v * this->kStepBytes);
      Scores::partial(s[v], st.q, f[v]);
    }
#pragma unroll
    for (int v = 0; v < N; ++v) {
      Scores::finish(*this, s[v]);
      dp[v] = this->head_sum(dp[v]);
    }
#pragma unroll
    for (int v = 0; v < N; ++v) {
      bool part[kMaps];   // by the bias: the row's lse may be NaN
#pragma unroll
      for (int m = 0; m < kMaps; ++m) part[m] = active[v];
      if constexpr (kBucket) {
        A b[kMaps];
        Bias::get(b, tab + v * GEO::kHeads * Bias::kBytes);
#pragma unroll
        for (int m = 0; m < kMaps; ++m) {
          part[m] = part[m] && b[m] != neg_inf<A>();
          s[v][m] += b[m];
        }
      }
      A g[kMaps], w = A(0);
#pragma unroll
      for (int m = 0; m < kMaps; ++m) {
        const A c = m == 0 ? A(1) : -st.lam;
        const A p = part[m] ? gk_exp2(s[v][m] - st.lse2[m]) * c : A(0);
        w += p;
        g[m] = p * (dp[v] - st.delta[m]);
        if (!part[m] || (kBucket && p == A(0))) g[m] = A(0);   // a masked row may hold anything
      }
      if (active[v] && st.ln.first) {
        EdgePair<A>* at = pd + ((unsigned long long)(pos + v) * (unsigned)Hp + st.ln.head * kMaps);
#pragma unroll
        for (int m = 0; m < kMaps; ++m) at[m] = EdgePair<A>{w, g[m]};
      }
      const bool up = kMaps == 2 && Scores::upper(*this);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const A x = Scores::of_slot(g, i, up);
        if (!kBucket || x != A(0)) st.acc[i].axpy(x, f[v][i]);
      }
    }
  }
  __device__ __forceinline__ int lse_at(int lane) const { return this->kNodeScalarAt + lane * (kMaps * (int)sizeof(A) - GEO::SB); }
  __device__ __forceinline__ void stage_node(const State& st, unsigned buf, int lane, int node) const {
    this->stage_row(st.ln, buf, reinterpret_cast<const unsigned char*>(q + st.ln.off), node, this->rowb, true);
    this->stage_row(st.ln, buf + kRow, reinterpret_cast<const unsigned char*>(dout + st.ln.off), node, this->rowb, true);
#pragma unroll
    for (int m = 0; m < kMaps; ++m)
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const A* at = sums + ((long long)(kMaps - 1) * st.ln.head * this->D + (long long)m * this->D + st.ln.off) + j * (V / kPer);
        const unsigned char* from = reinterpret_cast<const unsigned char*>(at) + (unsigned long long)(unsigned)node * (kMaps * kPer * this->rowb);
#pragma unroll
        for (int i = 0; i < W; ++i)
          cp_async_slot<GEO::SB>(buf + (2 + m * kPer + j) * kRow + i * 32 * GEO::SB, from + (size_t)(i * this->slot_step()) * sizeof(A),
                                 this->has(st.ln, i));
      }
    cp_async_slot<kMaps * sizeof(A)>(buf + lse_at(lane), lse + ((long long)node * this->H + st.ln.head) * kMaps, true);
  }
  __device__ __forceinline__ void begin(State& st, unsigned buf, int lane) const {
    F ov[W];
    this->load_staged(st.q, buf);
    this->load_staged(st.gr, buf + kRow);
    begin_merge(st);
#pragma unroll
    for (int m = 0; m < kMaps; ++m) {
      lds(st.lse2[m], buf + lse_at(lane) + m * (int)sizeof(A));
      if constexpr (kPer == 1) {
        this->load_staged(ov, buf + (2 + m) * kRow);
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            Frag<A, V / kPer> half;
            frag_lds<A, GEO::SB>(half, buf + (2 + m * kPer + j) * kRow + i * 32 * GEO::SB);
#pragma unroll
            for (int k = 0; k < V / kPer / 2; ++k) ov[i].p[j * (V / kPer / 2) + k] = half.p[k];
          }
      }
      st.delta[m] = frag_dot<V, W>(st.gr, ov);   // this lane's part: summed in began()
    }
    const A c = scale * A(kLog2e);
#pragma unroll
    for (int i = 0; i < W; ++i) st.q[i].scale(c);
  }
  // t = dO . o in the order dO . v is formed: a node with one edge gets dp - t = 0 exactly
  __device__ __forceinline__ void began(State& st, int node, bool mine) const {
#pragma unroll
    for (int m = 0; m < kMaps; ++m) {
      const A d = this->head_sum(st.delta[m]);
      if (mine) {
        const bool none = st.lse2[m] == neg_inf<A>();   // nothing took part: every probability is zero, whatever dO holds
        st.delta[m] = none ? A(0) : d;
        if (m == 1 && st.ln.first) t2[(long long)node * this->H + st.ln.head] = st.delta[m];
        st.lse2[m] = none ? -neg_inf<A>() : st.lse2[m] * A(kLog2e);
      }
    }
  }
  __device__ __forceinline__ void store_row(const State& st, int node) const {
    F out[W];
#pragma unroll
    for (int i = 0; i < W; ++i) { out[i] = st.acc[i]; out[i].scale(scale); }
    this->store_row_slots(st.ln, dq + (long long)node * this->HD + st.ln.off, out);
  }
  __device__ __forceinline__ void zero_row(const State& st, long long n) const {
    this->zero_slots(st.ln, dq, n);
    if (kMaps == 2 && st.ln.first) t2[n * this->H + st.ln.head] = A(0);
  }
  static constexpr int kCarryElems = GEO::kAccs;
  __device__ __forceinline__ void begin_merge(State& st) const {
#pragma unroll
    for (int i = 0; i < W; ++i) st.acc[i].zero();
  }
  __device__ __forceinline__ void save_carry(const State& st, A* rec, int gl) const { this->save_acc(rec, gl, st.acc); }
  __device__ __forceinline__ void load_carry(Carry& c, const A* rec, int gl) const { this->load_acc_raw(c.x, rec, gl); }
  __device__ __forceinline__ void merge(State& st, const Carry& c) const {
#pragma unroll
    for (int i = 0; i < W; ++i) st.acc[i].add(c.x[i]);
  }
};

// Source side: the plain layer's sums over the transposed CSR with pairs (w, g), a head per map.  The scale is applied once per
// row, so that dT has the unscaled g; a weight or score gradient of zero is passed over, so that what takes no part, a position or one
// map of it, may have anything in its rows of q and dO.
template <class GEO>
struct TermsBwdSrc : GroupAttnBwdSrc<GEO, true> {
  using Base = GroupAttnBwdSrc<GEO, true>;
  using T = typename GEO::T;
  using A = typename GEO::A;
  using F = typename GEO::F;
  using State = typename Base::State;
  static constexpr int W = GEO::W, kRow = GEO::kRow;
  template <int N>
  __device__ __forceinline__ void fold(State& st, unsigned slot, unsigned tab, const bool (&)[N], unsigned,
                                       const int (&)[N]) const {
#pragma unroll
    for (int v = 0; v < N; ++v) {
      F fq[W], fg[W];
      this->load_staged(fq, slot + v * this->kStepBytes);
      this->load_staged(fg, slot + v * this->kStepBytes + kRow);
      A w, g;
      lds2(w, g, tab + v * GEO::kHeads * 2 * (int)sizeof(A));
      if (w != A(0)) {
#pragma unroll
        for (int i = 0; i < W; ++i) st.av[i].axpy(w, fg[i]);
      }
      if (g != A(0)) {   // zero alone where the other map takes part
#pragma unroll
        for (int i = 0; i < W; ++i) st.ak[i].axpy(g, fq[i]);
      }
    }
  }
  __device__ __forceinline__ void store_row(const State& st, int node) const {
    const long long at = (long long)node * this->HD + st.ln.off;
    F out[W];
#pragma unroll
    for (int i = 0; i < W; ++i) { out[i] = st.ak[i]; out[i].scale(this->scale); }
    this->store_row_slots(st.ln, this->dk + at, out);
    this->store_row_slots(st.ln, this->dv + at, st.av);
  }
};
template <class GEO>
struct TermsSumPairs : SumAttnPairs<GEO> {
  using Base = SumAttnPairs<GEO>;
  using T = typename GEO::T;
  using A = typename GEO::A;
  using F = typename GEO::F;
  using State = typename Base::State;
  using Rows = typename Base::Rows;
  A scale;
  __device__ __forceinline__ void fold(State& st, const Rows& r, unsigned tab) const {
    F fq, fg;
    frag_unpack<T, GEO::SB>(fq, r.q);
    frag_unpack<T, GEO::SB>(fg, r.g);
    A w, g;
    lds2(w, g, tab);
    if (w != A(0)) st.av[0].axpy(w, fg);
    if (g != A(0)) st.ak[0].axpy(g, fq);
  }
  __device__ __forceinline__ void store_row(State& st, int node) const {
    this->flush(st);
    const long long at = (long long)node * this->HD + st.ln.off;
    F out[1] = {st.sk[0]};
    out[0].scale(scale);
    this->store_row_slots(st.ln, this->dk + at, out);
    this->store_row_slots(st.ln, this->dv + at, st.sv);
  }
};

// ---------------------------------------------------------------------------------------
// sums by bucket: out[b, h] = sign * sum of x[j, h] over the rows j of bucket b (bucket null: all rows are bucket 0)
// ---------------------------------------------------------------------------------------
// A stream of `lanes` threads, one head each, adds a contiguous range of rows into a table of its own in shared memory, one row
// after the other; the streams' tables, and then the blocks', are added up in order.  No atomics: the same bits every time.  What takes
// the time is waiting for rows, as the private tables leave a few hundred threads per SM: kBatch rows are asked for at once, and the
// next ones before the last are added (4.5M edges, 4 heads, 128 buckets: 84 us with batches of four, none ahead).
struct BucketSum {
  const int32_t* bucket;
  const PlanHeader* hdr;      // the rows are positions: only those that a chunk covers count; null: all of them
  long long rows, row_stride; // stride in elements
  int col_stride, columns;    // columns (heads) of x
  int buckets, per, streams, lanes;   // per: columns of a block (blockIdx.y counts such blocks)
};
constexpr int kBatch = 16;
template <typename A>
__global__ void __launch_bounds__(256)
bucket_sum_kernel(const A* __restrict__ x, const BucketSum a, double* __restrict__ partial) {
  extern __shared__ uint4 gk_ring[];
  A* cells = reinterpret_cast<A*>(gk_ring);
  const int tid = threadIdx.x, stream = tid / a.lanes, col = tid - stream * a.lanes, c0 = blockIdx.y * a.per;
  const int cols = a.columns - c0 < a.per ? a.columns - c0 : a.per, size = a.buckets * a.per;
  long long lo = 0, hi = a.rows;
  if (a.hdr) {
    lo = a.hdr->cover_lo > 0 ? a.hdr->cover_lo : 0;
    hi = a.hdr->cover_hi < a.rows ? a.hdr->cover_hi : a.rows;
  }
  const long long all = (long long)gridDim.x * a.streams, each = hi > lo ? (hi - lo + all - 1) / all : 0;
  const bool works = stream < a.streams && col < cols;
  const long long j0 = lo + ((long long)blockIdx.x * a.streams + stream) * each, j1 = !works ? j0 : j0 + each < hi ? j0 + each : hi;
  const A* src = x + (long long)(c0 + (works ? col : 0)) * a.col_stride;
  int b0[kBatch], b1[kBatch];
  A g0[kBatch], g1[kBatch];
  const auto ask = [&](int (&b)[kBatch], A (&g)[kBatch], long long j) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const bool in = j + u < j1;
      b[u] = !in ? -1 : a.bucket ? __ldg(a.bucket + j + u) : 0;
      g[u] = in ? __ldg(src + (j + u) * a.row_stride) : A(0);
    }
  };
  ask(b0, g0, j0);
  for (int i = tid; i < a.streams * size; i += blockDim.x) cells[i] = A(0);
  __syncthreads();
  A* mine = cells + (size_t)stream * size + col;
  const auto add = [&](const int (&b)[kBatch], const A (&g)[kBatch]) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if ((unsigned)b[u] < (unsigned)a.buckets) mine[(size_t)b[u] * a.per] += g[u];
  };
  for (long long j = j0; j < j1; j += 2 * kBatch) {
    ask(b1, g1, j + kBatch);
    add(b0, g0);
    ask(b0, g0, j + 2 * kBatch);
    add(b1, g1);
  }
  __syncthreads();
  double* out = partial + (size_t)blockIdx.x * a.buckets * a.columns;
  for (int i = tid; i < size; i += blockDim.x) {
    const int b = i / a.per, c = i - b * a.per;
    if (c >= cols) continue;
    double s = 0;
    for (int k = 0; k < a.streams; ++k) s += (double)cells[(size_t)k * size + i];
    out[(size_t)b * a.columns + c0 + c] = s;
  }
}
// The blocks' partials of 8 cells per block of this kernel: 32 threads per cell take every 32nd block, then add up by halves.
template <typename T>
__global__ void __launch_bounds__(256)
bucket_total_kernel(const double* __restrict__ partial, int blocks, int cells, double sign, T* __restrict__ out) {
  __shared__ double s_part[32][9];
  const int c = threadIdx.x & 7, slice = threadIdx.x >> 3, i = blockIdx.x * 8 + c;
  double s = 0;
  if (i < cells) {
#pragma unroll 8
    for (int b = slice; b < blocks; b += 32) s += partial[(size_t)b * cells + i];
  }
  s_part[slice][c] = s;
  __syncthreads();
  const int lane = threadIdx.x & 31, cell = threadIdx.x >> 5;   // a warp per cell
  s = s_part[lane][cell];
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
  const int at = blockIdx.x * 8 + cell;
  if (lane == 0 && at < cells) out[at] = from_acc<T>((typename AccOf<T>::type)(sign * s));
}

constexpr int kSumSmem = 32 * 1024;             // of a block
constexpr int kMostBuckets = 16384;
// How a sum by bucket is launched.
struct BucketShape { int lanes, per, streams, blocks, col_blocks; };
inline BucketShape bucket_shape(long long rows, int columns, int buckets, int acc) {
  BucketShape s;
  s.lanes = 1;
  while (s.lanes < 32 && s.lanes < columns) s.lanes <<= 1;
  // a table that is too large goes with fewer columns per block
  while (s.lanes > 1 && (long long)s.lanes * buckets * acc > kSumSmem) s.lanes >>= 1;
  s.per = s.lanes < columns ? s.lanes : columns;
  const long long table = (long long)s.per * buckets * acc, fit = kSumSmem / table;
  s.streams = 256 / s.lanes;
  if (s.streams > fit) s.streams = fit < 1 ? 1 : (int)fit;
  s.col_blocks = (columns + s.per - 1) / s.per;
  // a stream has two batches at least, and the chip as many blocks as its SMs hold, over all blocks of columns: their tables are added up
  int per_sm = (int)(200 * 1024 / (s.streams * table + 1024)), threads = s.streams * s.lanes;
  per_sm = per_sm < 1 ? 1 : per_sm > 6 ? 6 : per_sm;
  if (per_sm * threads > 1024) per_sm = 1024 / threads;
  const long long want = rows / (2ll * kBatch * s.streams) + 1, most = per_sm * 148 / s.col_blocks + 1;
  s.blocks = (int)(want < most ? want : most);
  return s;
}
inline size_t bucket_sum_bytes(long long rows, int columns, int buckets, int acc) {
  return align_up((size_t)bucket_shape(rows, columns, buckets, acc).blocks * buckets * columns * sizeof(double));
}
template <typename T, typename A = typename AccOf<T>::type>
inline int run_bucket_sum(Arena& ar, const A* x, long long rows, long long row_stride, int col_stride, int columns, const int32_t* bucket,
                          int buckets, const PlanHeader* hdr, double sign, T* out, cudaStream_t st) {
  const BucketShape s = bucket_shape(rows, columns, buckets, (int)sizeof(A));
  double* partial = (double*)ar.take((size_t)s.blocks * buckets * columns * sizeof(double));
  if (ar.overflow) return GRAPHOP_ERR_WORKSPACE;
  const int smem = s.streams * s.per * buckets * (int)sizeof(A), threads = (s.streams * s.lanes + 31) / 32 * 32;
  static std::atomic<bool> configured[64];
  if (smem > 48 * 1024) GK_TRY(allow_smem(bucket_sum_kernel<A>, kMostBuckets * (int)sizeof(A) > kSumSmem ? kMostBuckets * (int)sizeof(A) : kSumSmem, configured));
  const BucketSum a{bucket, hdr, rows, row_stride, col_stride, columns, buckets, s.per, s.streams, s.lanes};
  bucket_sum_kernel<A><<<dim3(s.blocks, s.col_blocks), threads, smem, st>>>(x, a, partial);
  GK_LAUNCHED("bucket_sum");
  const int cells = buckets * columns;
  bucket_total_kernel<T><<<(cells + 7) / 8, 256, 0, st>>>(partial, s.blocks, cells, sign, out);
  GK_LAUNCHED("bucket_total");
  return GRAPHOP_OK;
}

// ---------------------------------------------------------------------------------------
// the layers
// ---------------------------------------------------------------------------------------
// What a call is about, either direction.  diff: H pairs of maps of D features each, else H heads of D.
template <typename T>
struct TermsCall {
  bool diff;
  const T *q, *k, *v, *table, *lam;
  const int32_t* bucket;
  int buckets;
  double scale;
  long long E, n_dst, n_src;
  int H, D;
  int maps() const { return diff ? 2 : 1; }
  int row_d() const { return diff ? 2 * D : D; }   // features of a head of v
  size_t node_bytes(long long n) const { return (size_t)n * H * row_d() * sizeof(T); }
};

// Defined in gk_terms_banded.cuh for bfloat16: the tensor-core kernels for dense-band graphs; GRAPHOP_ERR_UNSUPPORTED when the call is
// not one they take.
template <typename T>
inline int banded_terms_forward(const graphop_plan_t*, const TermsCall<T>&, T*, void*, void*, void*, size_t, cudaStream_t) {
  return GRAPHOP_ERR_UNSUPPORTED;
}
template <typename T>
inline int banded_terms_backward(const graphop_plan_t*, const graphop_plan_t*, const TermsCall<T>&, const void*, const void*, const T*, T*,
                                 T*, T*, T*, T*, void*, size_t, cudaStream_t) {
  return GRAPHOP_ERR_UNSUPPORTED;
}

// The geometry of a row of H heads of D elements of `elem` bytes: the plain layer's, but blocks of as many heads as divide their number,
// where that makes every lane own whole slots known at compile time.
inline GeoPick terms_geo(int H, int D, int elem) {
  const GeoPick p = pick_geo(H, D, elem, 16, false);
  if (p.LT || (H & (H - 1)) == 0) return p;
  GeoPick q = pick_geo(H & -H, D, elem, 16, false);   // the largest power of two in H
  if (!q.LT) return p;
  q.nhb = H / (q.G / q.L);
  return q;
}
// Carry levels of the walks of such rows, in whatever geometry of the two walkers they get.  Blocks that divide the number of heads may be
// many more than walk_bytes counts, each with records and their ids (8-byte elements, 47 heads of 8: 47 blocks of 4 lanes for 6 of 16 x 2
// slots; 6016 bytes of sums and 188 of ids for 6144 and 24).
inline size_t terms_walk_bytes(long long E, long long n_nodes, int H, int D, int elem, int accs, int stats) {
  const GeoPick p = terms_geo(H, D, elem);
  const size_t most = walk_bytes(E, n_nodes, H, D, elem, false, accs, stats);
  const size_t own = carry_bytes(tile_bound(E, n_nodes), p.nhb, (long long)accs * p.accs(elem) + stats * p.G, elem == 8 ? 8 : 4);
  return p.SB && own > most ? own : most;
}

template <typename T>
inline int terms_check(const TermsCall<T>& c, long long C, bool al, GeoPick* geo) {
  GK_TRY(check_sizes(C, c.E, c.n_dst, c.n_src, c.H, c.D));
  if ((long long)c.H * c.D >= (1LL << 23)) return GRAPHOP_ERR_INVALID_ARGUMENT;
  if (c.buckets < (c.diff ? 0 : 1)) return GRAPHOP_ERR_INVALID_ARGUMENT;
  if (c.buckets > kMostBuckets) return GRAPHOP_ERR_UNSUPPORTED;
  if (!is_pow2(c.D * (int)sizeof(T) / 16) || c.D * (int)sizeof(T) % 16) return GRAPHOP_ERR_UNSUPPORTED;
  if (!attention_shape_ok<T>(c.H, c.row_d(), al, geo)) return GRAPHOP_ERR_UNSUPPORTED;
  *geo = terms_geo(c.H, c.row_d(), sizeof(T));
  return GRAPHOP_OK;
}
inline bool aligned_to(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

template <typename T, int kMaps, bool kBucket>
inline int run_terms_forward(Arena& ar, const GraphView& g, const GeoPick& s, const TermsCall<T>& c, T* o, void* sums, void* lse,
                             cudaStream_t st) {
  return dispatch_geo<T, false, true>(s, [&](auto tag) -> int {
    TermsFwd<typename decltype(tag)::type, kMaps, kBucket> op;
    using A = typename decltype(op)::A;
    fill_geo(op, s, c.H, c.row_d());
    op.q = c.q; op.k = c.k; op.v = c.v; op.table = c.table; op.lam = c.lam; op.o = o; op.each = (A*)sums; op.lse = (A*)lse;
    op.scale = (A)c.scale; op.buckets = c.buckets;
    return launch_walk(ar, g, s, op, c.n_dst, tiles_near(2 * (long long)c.node_bytes(c.n_src)), st);
  });
}

template <typename T, class GS>
inline int terms_forward(const GS& gs, long long C, const TermsCall<T>& c, T* o, void* sums, void* lse, void* ws, size_t wsb,
                         cudaStream_t st) {
  using A = typename AccOf<T>::type;
  GeoPick s;
  const bool al = aligned16(c.q) && aligned16(c.k) && aligned16(c.v) && aligned16(o) && aligned16(sums);
  GK_TRY(terms_check(c, C, al, &s));
  if (c.n_dst == 0) return c.E ? GRAPHOP_ERR_INVALID_ARGUMENT : GRAPHOP_OK;
  if (!o || !lse || !aligned_to(lse, c.maps() * sizeof(A))) return GRAPHOP_ERR_INVALID_ARGUMENT;
  if (c.E == 0) {   // no edge anywhere
    GK_CUDA(cudaMemsetAsync(o, 0, c.node_bytes(c.n_dst), st));
    if (sums) GK_CUDA(cudaMemsetAsync(sums, 0, c.maps() * c.node_bytes(c.n_dst) / sizeof(T) * sizeof(A), st));
    const long long cells = c.n_dst * c.H * c.maps();
    fill_kernel<A><<<(unsigned)((cells + 255) / 256 < 4096 ? (cells + 255) / 256 : 4096), 256, 0, st>>>((A*)lse, neg_inf_host<A>(), cells);
    GK_LAUNCHED("fill");
    return GRAPHOP_OK;
  }
  if (!c.q || !c.k || !c.v || !gs.valid(true) || (c.diff && !c.lam) || (c.buckets && (!c.bucket || !c.table)))
    return GRAPHOP_ERR_INVALID_ARGUMENT;
  GK_TRY(check_ws(ws));
  if constexpr (std::is_same_v<GS, FromPlan>) {
    const int rc = banded_terms_forward<T>(gs.p, c, o, sums, lse, ws, wsb, st);
    if (rc != GRAPHOP_ERR_UNSUPPORTED) return rc;
  }
  Arena ar(ws, wsb);
  GraphView g;
  GK_TRY(gs(ar, c.n_dst, st, &g));
  g.eid = c.buckets ? c.bucket : nullptr;
  if (!c.diff) return run_terms_forward<T, 1, true>(ar, g, s, c, o, sums, lse, st);
  if (c.buckets) return run_terms_forward<T, 2, true>(ar, g, s, c, o, sums, lse, st);
  return run_terms_forward<T, 2, false>(ar, g, s, c, o, sums, lse, st);
}

template <typename T, int kMaps, bool kBucket, class A>
inline int run_terms_dst(Arena& ar, const GraphView& g, const GeoPick& s, const TermsCall<T>& c, const void* sums, const void* lse,
                         const T* dout, EdgePair<A>* pd, int Hp, A* t2, T* dq, cudaStream_t st) {
  return dispatch_geo<T, false, true>(s, [&](auto tag) -> int {
    TermsBwdDst<typename decltype(tag)::type, kMaps, kBucket> op;
    fill_geo(op, s, c.H, c.row_d());
    op.q = c.q; op.k = c.k; op.v = c.v; op.table = c.table; op.lam = c.lam; op.sums = (const A*)sums; op.dout = dout; op.lse = (const A*)lse;
    op.pd = pd; op.t2 = t2; op.dq = dq; op.scale = (A)c.scale; op.Hp = Hp; op.buckets = c.buckets;
    return launch_walk(ar, g, s, op, c.n_dst, tiles_near(2 * (long long)c.node_bytes(c.n_src)), st);
  });
}
// dk and dv, a head per map of D features
template <typename T, class A>
inline int run_terms_src(Arena& ar, const GraphView& g, const TermsCall<T>& c, const T* dout, const EdgePair<A>* pd, int Hp, T* dk,
                         T* dv, cudaStream_t st) {
  const int H = c.H * c.maps(), D = c.D;
  const long long table = (long long)c.node_bytes(c.n_dst);
  const GeoPick s = terms_geo(H, D, sizeof(T));
  const auto ring = [&](int only, int most) -> int {
    return dispatch_geo<T, false, true>(s, [&](auto tag) -> int {
      TermsBwdSrc<typename decltype(tag)::type> op;
      fill_geo(op, s, H, D);
      op.q = c.q; op.k = nullptr; op.v = nullptr; op.dout = dout; op.stat = nullptr; op.pd = pd; op.dk = dk; op.dv = dv;
      op.scale = (A)c.scale; op.Hp = Hp;
      return launch_walk(ar, g, s, op, c.n_src, most, st, only);
    });
  };
  if constexpr (kSumsByRegister<T>) {
    const GeoPick p = pick_sum_geo(H, D, sizeof(T), 16);
    return choose_walker(ar, g, 2, table, p.nhb, c.n_dst, st, [&](bool sums, int only, int most) -> int {
      if (!sums) return ring(only, most);
      return dispatch_sum_geo<T, false>(p, [&](auto tag) -> int {
        TermsSumPairs<typename decltype(tag)::type> op;
        fill_geo(op, p, H, D);
        op.q = c.q; op.dout = dout; op.pd = pd; op.dk = dk; op.dv = dv; op.Hp = Hp; op.scale = (A)c.scale;
        op.wide_scalars = wide_scalars(p, pd, Hp, 2 * (int)sizeof(A));
        return launch_walk(ar, g, p, op, c.n_src, most, st, only);
      });
    });
  } else {
    return ring(-1, tiles_near(2 * table));
  }
}

// sums: what the forward left in `sums`, or its output where that is the accumulator type.  The transposed CSR carries edge ids: for each of its positions the row-CSR
// position of the same edge.
template <typename T, class GS>
inline int terms_backward(const GS& gs_r, const GS& gs_c, bool has_eid_t, long long C, long long Ct, const TermsCall<T>& c, const void* sums,
                          const void* lse, const T* dout, T* dq, T* dk, T* dv, T* d_table, T* d_lam, void* ws, size_t wsb,
                          cudaStream_t st) {
  using A = typename AccOf<T>::type;
  GeoPick s;
  const bool al = aligned16(c.q) && aligned16(c.k) && aligned16(c.v) && aligned16(sums) && aligned16(dout) && aligned16(dq) &&
                  aligned16(dk) && aligned16(dv);
  GK_TRY(terms_check(c, C, al, &s));
  if (Ct < 0 || (c.n_dst && !dq) || (c.n_src && (!dk || !dv)) || (c.buckets && !d_table) || (c.diff && !d_lam))
    return GRAPHOP_ERR_INVALID_ARGUMENT;
  const int columns = c.H * c.maps();
  if (c.E == 0) {   // no edge: every gradient is zero
    if (c.n_dst) GK_CUDA(cudaMemsetAsync(dq, 0, c.node_bytes(c.n_dst), st));
    if (c.n_src) GK_CUDA(cudaMemsetAsync(dk, 0, c.node_bytes(c.n_src), st));
    if (c.n_src) GK_CUDA(cudaMemsetAsync(dv, 0, c.node_bytes(c.n_src), st));
    if (c.buckets) GK_CUDA(cudaMemsetAsync(d_table, 0, (size_t)c.buckets * columns * sizeof(T), st));
    if (c.diff) GK_CUDA(cudaMemsetAsync(d_lam, 0, (size_t)c.H * sizeof(T), st));
    return GRAPHOP_OK;
  }
  if (!has_eid_t || !gs_r.valid(true) || !gs_c.valid(true) || !c.q || !c.k || !c.v || !sums || !lse || !dout || !c.n_dst || !c.n_src ||
      (c.diff && !c.lam) || (c.buckets && (!c.bucket || !c.table)) || !aligned_to(lse, c.maps() * sizeof(A)))
    return GRAPHOP_ERR_INVALID_ARGUMENT;
  GK_TRY(check_ws(ws));
  if constexpr (std::is_same_v<GS, FromPlan>) {
    const int rc = banded_terms_backward<T>(gs_r.p, gs_c.p, c, sums, lse, dout, dq, dk, dv, d_table, d_lam, ws, wsb, st);
    if (rc != GRAPHOP_ERR_UNSUPPORTED) return rc;
  }
  Arena ar(ws, wsb);
  const int Hp = stat_heads(columns, (int)sizeof(A));
  auto* pd = (EdgePair<A>*)ar.take((size_t)c.E * Hp * sizeof(EdgePair<A>));   // survives both passes
  A* t2 = c.diff ? (A*)ar.take((size_t)c.n_dst * c.H * sizeof(A)) : nullptr;
  const size_t mark = ar.used;
  {
    GraphView g;
    GK_TRY(gs_r(ar, c.n_dst, st, &g));
    g.eid = c.buckets ? c.bucket : nullptr;
    if (!c.diff) GK_TRY((run_terms_dst<T, 1, true>(ar, g, s, c, sums, lse, dout, pd, Hp, t2, dq, st)));
    else if (c.buckets) GK_TRY((run_terms_dst<T, 2, true>(ar, g, s, c, sums, lse, dout, pd, Hp, t2, dq, st)));
    else GK_TRY((run_terms_dst<T, 2, false>(ar, g, s, c, sums, lse, dout, pd, Hp, t2, dq, st)));
    if (c.buckets)
      GK_TRY((run_bucket_sum<T>(ar, &pd->ds, c.E, 2ll * Hp, 2, columns, c.bucket, c.buckets, g.hdr, 1.0, d_table, st)));
    if (c.diff) GK_TRY((run_bucket_sum<T>(ar, t2, c.n_dst, c.H, 1, c.H, nullptr, 1, nullptr, -1.0, d_lam, st)));
  }
  ar.used = mark;
  GraphView g;
  GK_TRY(gs_c(ar, c.n_src, st, &g));
  return run_terms_src<T>(ar, g, c, dout, pd, Hp, dk, dv, st);
}

// bytes of workspace of either direction, by the walkers
inline size_t terms_bytes(bool diff, bool backward, long long E, long long n_nodes, int H, int D, int buckets, int elem, int index_bytes) {
  const size_t acc = elem == 8 ? 8 : 4;
  const int maps = diff ? 2 : 1, columns = H * maps, row_d = D * maps;
  size_t need = graph_bytes(E, n_nodes, index_bytes);
  if (!backward) return need + terms_walk_bytes(E, n_nodes, H, row_d, elem, maps, 2 * maps) + kAlign;
  need += align_up((size_t)E * stat_heads(columns, (int)acc) * 2 * acc);
  if (diff) need += align_up((size_t)n_nodes * H * acc) + bucket_sum_bytes(n_nodes, H, 1, (int)acc);
  if (buckets) need += bucket_sum_bytes(E, columns, buckets, (int)acc);
  const size_t dst = terms_walk_bytes(E, n_nodes, H, row_d, elem, 1, 0), src = terms_walk_bytes(E, n_nodes, columns, D, elem, 2, 0);
  return need + (dst > src ? dst : src) + kAlign;
}

}  // namespace gk
