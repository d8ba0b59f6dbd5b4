// g2v_counts.h -- whole-number helpers of the operators' kernels whose arguments
// go up to 2^31 - 1: nothing in them leaves int.  Plain C++: usable on both sides.
#pragma once

namespace g2v {

// pieces of `size` elements that n elements take (n + size - 1 may pass 2^31 - 1)
constexpr int pieces(int n, int size) { return n / size + (n % size != 0); }

// the same for a size of 2^log2, without a division
constexpr int pieces_log2(int n, int log2) {
  return (n >> log2) + ((n & ((1 << log2) - 1)) != 0);
}

// rows v in [0, V) with v % buckets == b
constexpr int rows_of_bucket(int V, int b, int buckets) {
  return V > b ? pieces(V - b, buckets) : 0;
}

}  // namespace g2v
