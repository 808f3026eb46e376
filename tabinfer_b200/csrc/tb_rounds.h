// tb_rounds.h -- the rounds in which several producer warps fill one pipeline of tiles, as plain
// C++: the kernel runs them with its barrier and copies, a host program with threads.
#pragma once
#ifdef __CUDACC__
#define TB_ROUNDS __host__ __device__ __forceinline__
#else
#define TB_ROUNDS inline
#endif

// One producer's walk over its tiles.  Every producer makes the same walk and meets the others
// at sync() once a tile.  have, next, after: whether there is a first, second and third tile.
//   publish(it + 1)   tells the others of the next tile
//   sync(dead)        the meeting; true when one of them has given up: all leave then
//   ahead()           looks at the tile after the next, true when another one follows
//   tile(it, next)    does tile it; false when a wait in it gave up
// A producer that gives up meets the others once more, for they come to the next tile's meeting,
// and not behind the last tile, where they come to none: each waits as often as the others.
template <class Publish, class Sync, class Ahead, class Tile>
TB_ROUNDS void producer_rounds(bool have, bool next, bool after, Publish publish, Sync sync, Ahead ahead, Tile tile)
{
    for (int it = 0; have; it++) {
        if (next) publish(it + 1);
        if (sync(false)) return;
        const bool later = after && ahead();
        if (!tile(it, next)) {
            if (next) sync(true);
            return;
        }
        have = next;
        next = after;
        after = later;
    }
}
