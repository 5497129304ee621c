// Plain C++, so that the host can check it too.
#pragma once

#include <cstdint>

#ifdef __HIPCC__
#define T2T_HOST_DEVICE __host__ __device__
#else
#define T2T_HOST_DEVICE
#endif

namespace t2t {

// Which pieces of a cache (kPiece positions each) the new rows of one sequence
// read: their causal range, or with a window and no grant words the hull of
// their windows (and of sinks behind it) and, before it, the hull of their
// sinks.  Piece i < count is piece at(i) of the cache.
template <int kPiece>
struct PieceRange {
  int sink0 = 0, sinks = 0, near0 = 0, count = 0;

  // rows tokens at q_pos, documents from q_start (NULL: no sinks); window 0:
  // none, or whole it has no effect
  T2T_HOST_DEVICE PieceRange(const int32_t* q_pos, const int32_t* q_start, int rows, int keys,
                             int window, int n_sinks) {
    int near_lo = 0x7fffffff, near_hi = -1, sink_lo = 0x7fffffff, sink_hi = -1;
    for (int t = 0; t < rows; ++t) {
      const int p = q_pos[t], last = least(p, keys - 1);
      if (last < 0) continue;
      const int64_t lo = window > 0 ? most((int64_t)p - window + 1, (int64_t)0) : 0;
      if (lo <= last) {
        near_lo = least(near_lo, (int)lo / kPiece);
        near_hi = most(near_hi, last / kPiece);
      }
      if (q_start) {
        const int64_t s = q_start[t], e = least(s + n_sinks - 1, (int64_t)last);
        if (e >= 0 && s <= e) {
          sink_lo = least(sink_lo, (int)most(s, (int64_t)0) / kPiece);
          sink_hi = most(sink_hi, (int)e / kPiece);
        }
      }
    }
    if (near_hi >= 0) {
      // (a row past the cache has sinks but no window here: they may lie behind
      // the windows' hull, which then ends with them)
      near_hi = most(near_hi, sink_hi);
      sink_hi = least(sink_hi, near_lo - 1);  // (the hull holds the others)
      near0 = near_lo;
      count = near_hi - near_lo + 1;
    }
    if (sink_lo <= sink_hi) {
      sink0 = sink_lo;
      sinks = sink_hi - sink_lo + 1;
      count += sinks;
    }
  }
  T2T_HOST_DEVICE int at(int i) const { return i < sinks ? sink0 + i : near0 + i - sinks; }

 private:
  template <typename T>
  T2T_HOST_DEVICE static T least(T a, T b) { return a < b ? a : b; }
  template <typename T>
  T2T_HOST_DEVICE static T most(T a, T b) { return a > b ? a : b; }
};

}  // namespace t2t
