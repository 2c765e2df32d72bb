// The merge's reading of a span, on the host (see test_paged_spans.py): 0 where every case holds, else the number of one that does not.
#include "paged_common.cuh"

int main() {
    const int parts[] = {1, 2, 74, 148, 65536}, words[] = {-2147483647 - 1, -2147483647, -65536, -1, 0, 1, 2, 73, 74, 147, 148, 65535, 65536, 2147483646, 2147483647};
    int id = 0;
    for (int n : parts)
        for (int first : words)
            for (int last : words) {
                ++id;
                const int got = smla::span_parts(first, last, n);
                const bool inside = first >= 0 && first < n && last >= 0 && last < n;
                if (got != (inside && last >= first ? last - first + 1 : 0)) return 1 + id % 200;
                // records [2 first, 2 (first + got)) of 2 n
                if (got > 0 && (first < 0 || (long long)first + got > n)) return 1 + id % 200;
            }
    return 0;
}
