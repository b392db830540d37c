// Where the copies of a CTA pair stand when a wait has run out.
//
// Both CTAs of a pair fill a ring of stages in the same order, each with copies of its own; the bytes of both are counted on the first CTA's barrier of
// the stage, which opens for its first CTA's arrival and completes with the last byte.  A CTA that gives up has issued the copies of the first n blocks,
// its peer of the first m: the barriers of the blocks between are short of bytes, and nobody can wait for the copies that are under way on them.
// So the one that is behind issues what it lacks -- no more than a ring of blocks, into stages that the MMAs have given back, or the other could not
// have issued them -- and the first CTA waits for the blocks of the last ring, after which no copy is under way in either.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define NNCV_BOTH __host__ __device__ __forceinline__
#else
#define NNCV_BOTH inline
#endif

namespace nncv_b200 {
namespace pair_copies {

struct Spot { uint32_t stage, parity; };   // of a block: its stage, and the parity of its barrier's phase
NNCV_BOTH Spot spot_of(long long block, int stages) { return {(uint32_t)(block % stages), (uint32_t)(block / stages) & 1u}; }
NNCV_BOTH long long meet_at(long long mine, long long theirs) { return mine > theirs ? mine : theirs; }
NNCV_BOTH long long wait_from(long long end, int stages) { return end > stages ? end - stages : 0; }   // the blocks before are complete

}  // namespace pair_copies
}  // namespace nncv_b200
#undef NNCV_BOTH
