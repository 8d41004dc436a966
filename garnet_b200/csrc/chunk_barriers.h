// The named barriers between the warps of a tile of chunk attention (attn_chunk_tc.cu): who comes to them, and when.  Plain arithmetic,
// without CUDA headers.
//
// A named barrier counts arrivals, not warps: one that came twice before the others came once would complete it for nobody, and whoever
// waits there has no time limit.  So no warp may come to a barrier again before its last phase is complete, also when a wait in shared
// memory (all of which have a limit) gave up and the data that it waited for will never be there.  Two sets of barriers, for even and odd
// steps:
//   scores(i)  the scout arrives, the softmax waits;
//   P(i)       the softmax arrives, the MMA issuer and the scout wait.
// The scout passes the scores of step i on behind P(i - 2), whatever became of its own wait: the softmax comes to P(i) behind
// scores(i), so P(i - 2) is complete by then, and to scores(i + 2) behind P(i), to which the softmax came behind scores(i).  The
// issuer takes P(i) in turn, waiting for it.
#pragma once

namespace gb200 {

constexpr int kScoresThreads = 32 + 128;      // scout, softmax
constexpr int kWeightsThreads = 128 + 32 + 32;   // softmax, issuer, scout

// The scout of a tile of `steps` steps: two more for P V of the last two.
template <typename TakeP, typename Wait, typename Pass>
#if defined(__CUDACC__)
__device__ __forceinline__
#else
inline
#endif
void chunk_scout(int steps, TakeP take_p, Wait wait, Pass pass)
{
    for (int i = 0; steps && i < steps + 2; ++i) {
        if (i >= 2) take_p(i - 2);
        wait(i);
        pass(i);
    }
}

}  // namespace gb200
