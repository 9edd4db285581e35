/* How the warps of a group go through work items together.  Plain C++ as well as device
 * code, so that a host test can run it with threads for warps.
 *
 * next(i) waits for item i and says whether this warp has it: false past the last item and
 * once a bounded wait of its has run out, which one warp's may and another's, a moment
 * later, not.  work(i) holds barriers of the whole group, without a limit, so no warp may
 * leave while another goes on: any(p) tells every warp of the group whether p holds for one
 * of them, and they leave together. */
#ifndef GLINT_B200_ITEM_LOOP_H_
#define GLINT_B200_ITEM_LOOP_H_

#ifdef __CUDACC__
#define GLINT_ITEM_LOOP_FN __device__ __forceinline__
#else
#define GLINT_ITEM_LOOP_FN inline
#endif

namespace glint {

template <class Next, class Any, class Work>
GLINT_ITEM_LOOP_FN void item_loop(Next &&next, Any &&any, Work &&work)
{
    for (int i = 0;; ++i) {
        const bool have = next(i);
        if (any(!have))
            return;
        work(i);
    }
}

} // namespace glint

#endif
