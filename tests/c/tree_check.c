/* ec_tree.h on the host: the checks of a sequence's numbers against sums in 64
 * bits, over every combination of edge values. */
#include "ec_tree.h"

#include <limits.h>
#include <stdio.h>

int main(void)
{
    const int v[] = {INT_MIN, INT_MIN + 1, -65, -1, 0, 1, 2, 3, 4, 63, 64, 65, 99, 100, 101, INT_MAX - 1, INT_MAX};
    const int n = sizeof v / sizeof *v;
    long seen = 0, bad = 0;
    for (int c = 0; c < n; c++)
        for (int m = 0; m < n; m++) {
            if (v[c] < 1 || v[m] < 0 || v[m] > v[c]) continue;
            EcTreeBatch t = {1, 64, 0, 0, 0, 0, 3, v[c], v[m]};
            for (int i = 0; i < n; i++)
                for (int j = 0; j < n; j++)
                    for (int k = 0; k < n; k++) {
                        t.slot = &v[i], t.past = &v[j], t.nodes = &v[k];
                        EcTreeSeq s = ec_tree_seq(&t, 0);
                        int want = v[i] >= 0 && v[i] < 3 && v[k] >= 0 && v[k] <= 64 && v[j] >= 0 && v[j] <= v[m] &&
                                   (long long)v[j] + v[k] <= v[c];
                        int rows = v[k] >= 0 && v[k] <= 64 ? v[k] : 64;
                        bad += ec_tree_seq_ok(&t, s) != want || ec_tree_rows(&t, s) != rows;
                        seen++;
                    }
        }
    for (int i = 0; i < 64; i++)
        for (int j = 0; j < n; j++) bad += ec_tree_parent_ok(v[j], i) != (v[j] >= -1 && v[j] < i), seen++;
    for (int p = 0; p < 12; p++)
        for (int q = 0; q < 12; q++)
            for (int a = 0; a < 6; a++)
                for (int b = 0; b < 6; b++) {
                    int want = 0;
                    for (int x = p; x < p + a; x++) want |= x >= q && x < q + b;
                    EcTreeSeq s = {1, p, a}, o = {1, q, b}, other = {2, q, b};
                    bad += ec_tree_clash(s, o) != want || ec_tree_clash(s, other);
                    seen++;
                }
    printf("%ld checks, %ld wrong\n", seen, bad);
    return bad != 0;
}
