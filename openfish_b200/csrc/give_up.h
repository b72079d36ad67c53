// give_up.h -- what a block of the matrix kernels has to see land before it ends, once one of its waits has run out: plain C++, so that it
// can be tried without a GPU.
//
// Whose wait that was says nothing about what is under way: a warp all of whose own waits were answered may have issued copies or
// products that another one has stopped waiting for.  So the block decides, by its common flag and behind its last barrier.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define OF_HD __host__ __device__ __forceinline__
#else
#define OF_HD inline
#endif

// The copies of a ring of stages that two blocks fill together (or one: mine == theirs).  Step i goes to stage i % ring; the bytes of both
// blocks count at the first block's barrier of the stage, where the first block announces all of them when it issues its own.  This block (the first) has
// issued `mine` steps, the other one `theirs`; neither is more than a ring ahead of what has been read.
//   announce(stage)        this block announces the other one's bytes, of a step that it has not come to itself
//   forgo(stage)           takes the other one's bytes, which will not come, off what has been announced
//   landed(stage, parity)  waits, with a limit, until what has been announced of that phase is there
template <class Announce, class Forgo, class Landed>
OF_HD void land_copies(int mine, int theirs, int ring, Announce announce, Forgo forgo, Landed landed) {
    const int all = mine > theirs ? mine : theirs;
    for (int i = all > ring ? all - ring : 0; i < all; ++i) {
        if (i >= mine) announce(i % ring);
        if (i >= theirs) forgo(i % ring);
        landed(i % ring, (uint32_t)(i / ring) & 1u);
    }
}
