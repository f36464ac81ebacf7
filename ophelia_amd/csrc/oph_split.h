// How an axis that several workgroups share is cut, for device code and host programs alike (no HIP in here).
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define OPH_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define OPH_HOST_DEVICE inline
#endif

namespace ophseq {

struct Span { int beg, end; };                 // elements beg..end-1; empty: beg == end

// Piece `split` of `nsplit` of an axis of n elements, in whole tiles of `tile`; !live: the empty span at its beginning.  Pieces are rounded up to
// tiles, so that the last ones of many may begin behind the axis: they are empty and lie at its end, 0 <= beg <= end <= n always holds.  64 bits,
// since the last piece's end, rounded up, can pass n by nsplit tiles, and n goes up to the last 32-bit numbers.
OPH_HOST_DEVICE Span split_span(int n, int tile, int nsplit, int split, bool live) {
    const int tiles = n / tile + (n % tile != 0);
    const int64_t per = (int64_t)((tiles + nsplit - 1) / nsplit) * tile, first = split * per;
    const int64_t beg = first < n ? first : n, end = beg + per < n ? beg + per : n;
    return Span{(int)beg, (int)(live ? end : beg)};
}

// Where lane `lane` of a tile that begins at `first` finds its element's flag: at the element, or at the span's last one for what lies behind it;
// -1: the tile holds nothing of the span, nothing may be read.
OPH_HOST_DEVICE int flag_index(int first, int lane, int end) {
    return first >= end ? -1 : first + lane < end ? first + lane : end - 1;
}

}  // namespace ophseq
