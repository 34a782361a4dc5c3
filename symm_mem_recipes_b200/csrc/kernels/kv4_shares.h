// Who has which tiles of a decode step's attention over a 4-bit cache, and where a head that was cut left its pieces.  Shared by
// the kernels that leave and join them and by a check on the host.
#pragma once

#ifdef __CUDACC__
#define SMR_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define SMR_HOST_DEVICE inline
#endif

namespace smr {
namespace kv4 {

constexpr int kWarps = 4;      // of an attention CTA

// The list's tiles among the warps: the first `more` of them have one tile more than the others.  (One 32-bit division; with
// tiles * w / warps in 64 bits the second kernel spent 20 us on divisions.)
struct Shares {
  int tiles, each, more;
  SMR_HOST_DEVICE Shares(int tiles, int warps) : tiles(tiles), each(tiles / warps), more(tiles - each * warps) {}
  SMR_HOST_DEVICE int first(int w) const { return w * each + (w < more ? w : more); }
  SMR_HOST_DEVICE int warp_of(int tile) const {
    const int of_more = more * (each + 1);
    return tile < of_more ? tile / (each + 1) : more + (tile - of_more) / each;      // each > 0 where a tile is behind those
  }
};

// The pieces of a head whose tiles are [s0, s1) of the list: one of every CTA that has some, at the first of its warps that does
// (warps that ended in the head joined theirs), and one more of the last warp, where that went on to another head and is not
// the first itself.  A warp has two places, the second for a head that is not its first.
struct HeadCut {
  Shares shares;
  int s0, wa, wb, ctas, count;
  bool finished;      // by one CTA
  SMR_HOST_DEVICE HeadCut(const Shares& shares, int s0, int s1)
      : shares(shares), s0(s0), wa(shares.warp_of(s0)), wb(shares.warp_of(s1 - 1)) {
    const int ca = wa / kWarps, cb = wb / kWarps, lead = wa > cb * kWarps ? wa : cb * kWarps;
    const bool ends = shares.first(wb + 1) == s1;
    ctas = cb - ca + 1;
    count = ctas + (!ends && wb != lead ? 1 : 0);
    finished = wa == wb || (ca == cb && ends);
  }
  SMR_HOST_DEVICE int place(int k) const {
    const int w = k == 0 ? wa : k < ctas ? (wa / kWarps + k) * kWarps : wb;
    return 2 * w + (shares.first(w) < s0 ? 1 : 0);
  }
};

// What a warp ends with: a head that it does not finish by itself.
struct FinalPiece {
  int head;
  bool whole, last;      // has the head's first tile, its last one
  int slot;              // of its two places
};
constexpr int kNoPiece = -1, kNoTiles = -2;

// The CTA's warps [w0, return) end in the head of warp w0; `last`: one of them has the head's last tile.
SMR_HOST_DEVICE int run_of(const FinalPiece* final_of, int w0, bool& last) {
  const int head = final_of[w0].head;
  last = final_of[w0].last;
  int w1 = w0 + 1;
  for (; w1 < kWarps && (final_of[w1].head == head || final_of[w1].head == kNoTiles); ++w1)
    if (final_of[w1].head == head) last = final_of[w1].last;
  return w1;
}

}  // namespace kv4

// 0 if every tile of every head (tiles[i] of head i, none for an idle one) reaches the output exactly once: heads that a warp or a CTA
// finishes, and the pieces that the second kernel finds where the first one left them.
int check_kv4_cuts(const int* tiles, int heads, int ctas);

}  // namespace smr
