// Which key tiles a query tile reads under a sliding window with sinks (query i sees key j <= i where i - j < window or
// j < sinks): shared by the host schedule, which cuts them into pieces, and the kernel, which walks a piece's. No includes
// and plain C++ but for the two qualifiers, so that a host compiler takes it as well.
#pragma once

namespace miattn {

// Of the segment's key tiles (BK keys each) up to a query tile's last row those that hold neither a sink nor a key within its
// first row's window are left out. The n others are numbered from 0.
struct Band {
  int ts, jump, n;
};

// Query rows row0 .. q_end - 1.
__host__ __device__ inline Band band_of(int row0, int q_end, int window, int sinks, int BK) {
  const int first = row0 - window + 1;
  const int tw = first > 0 ? first / BK : 0;  // first tile of the window
  const int s = ((sinks < q_end ? sinks : q_end) + BK - 1) / BK;
  Band b;
  b.ts = s < tw ? s : tw;
  b.jump = tw - b.ts;
  b.n = (q_end + BK - 1) / BK - b.jump;
  return b;
}

// The segment's tile that number t is: the sinks' tiles, then the window's.
__host__ __device__ inline int band_tile(int t, int ts, int jump) { return t < ts ? t : t + jump; }

}  // namespace miattn
