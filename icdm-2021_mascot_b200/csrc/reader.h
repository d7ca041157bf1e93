// What a warp that reads accumulators and scales out of shared buffers may still do after one of its waits has run out (row_product.cu).
//
// A buffer is handed back by arriving on a barrier, and whoever fills it again counts arrivals without seeing whose they are.  An arrival of a
// reader that no longer waits would stand in for one that has not read yet, and what that one still needs would be
// overwritten: finite scores, and wrong ones.  So a reader that gave up arrives nowhere any more, and whatever it stores is NaN, other warps' lanes
// included, since the scales it multiplies by need not be there.  The others run out of their own waits then, one after the other.
// Free of CUDA calls, so that a host-only test can drive it.
#pragma once

#ifdef __CUDACC__
#define READER_FN __host__ __device__ __forceinline__
#else
#define READER_FN inline
#endif

namespace mascot {

class Reader {
public:
    READER_FN bool ok() const { return ok_; }
    READER_FN void waited(bool came) { ok_ = ok_ && came; }                        // for a warp: the same in all its lanes
    template <class Arrive> READER_FN void hand_back(Arrive arrive) const { if (ok_) arrive(); }
    READER_FN float factor(float scale) const { return ok_ ? scale : __builtin_nanf(""); }
private:
    bool ok_ = true;
};

}  // namespace mascot
