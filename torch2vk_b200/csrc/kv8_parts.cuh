// Records that the decode kernel leaves for its joining kernel: which CTAs hold parts of a unit.  Plain C++ too.
#pragma once

#ifdef __CUDACC__
#define T2C_HOST_DEVICE __host__ __device__
#else
#define T2C_HOST_DEVICE
#endif

namespace t2c {

// Parts of a unit whose tiles lie in CTAs first .. last, of `ctas` CTAs and with at most `most` parts a unit.  0 for a
// record that names anything else: a CTA whose wait ran out leaves the records of its units unwritten, so they hold what
// the workspace held, and no index may be made of that.
T2C_HOST_DEVICE inline int kv8_part_count(int first, int last, int ctas, int most) {
    if (first < 0 || last < first || last >= ctas) return 0;
    return last - first < most ? last - first + 1 : 0;
}

}  // namespace t2c
