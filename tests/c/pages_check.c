/* ec_pages.h on the host: the page of a row against a division, for every page size up
 * to 4096 and the edges of others, and the checks of a sequence's numbers against sums in
 * 64 bits, over combinations of edge values. */
#include "ec_pages.h"

#include <limits.h>
#include <stdio.h>

int main(void)
{
    long seen = 0, bad = 0;
    for (long i = 1; i <= 4096 + 400; i++) {
        const long far[] = {4097, 5000, 65535, 65536, 65537, 1000003, (1L << 30) - 1, 1L << 30, (1L << 30) + 1, INT_MAX - 1, INT_MAX};
        const long page = i <= 4096 ? i : i <= 4107 ? far[i - 4097] : (i - 4107) * 5000011L;
        EcPageBatch t = {1, 1, 0, 0, 0, 1, 1, (int)page, 1, 1, 0, 0};
        ec_pages_divide(&t);
        for (long q = 0; q <= INT_MAX / page; q = q < 70 ? q + 1 : q * 3 + 1)
            for (long d = -1; d <= 1; d++) {
                const long p = q * page + d;
                if (p < 0 || p > INT_MAX) continue;
                bad += ec_page_of(&t, (int)p) != (int)(p / page), seen++;
            }
        for (long p = INT_MAX; p > INT_MAX - 3; p--) bad += ec_page_of(&t, (int)p) != (int)(p / page), seen++;
    }
    const int v[] = {INT_MIN, INT_MIN + 1, -65, -1, 0, 1, 2, 9, 10, 11, 99, 100, 101, (1 << 30) - 1, 1 << 30, (1 << 30) + 1, INT_MAX - 1, INT_MAX};
    const int n = sizeof v / sizeof *v;
    for (int m = 0; m < 3; m++)
        for (int r = 0; r < 3; r++)
            for (int i = 0; i < n; i++)
                for (int j = 0; j < n; j++)
                    for (int k = 0; k < n; k++)
                        for (int x = 0; x < n; x++) {
                            const int M = m == 0 ? 1 : m == 1 ? 10 : 1 << 22, rows = r == 0 ? 1 : r == 1 ? 100 : 1 << 30;
                            const int start[2] = {v[i], v[j]};
                            EcPageBatch t = {1, M, start, &v[k], 0, 1, 1, 1, 1, rows, 0, 0};
                            const EcPageSeq s = ec_page_seq(&t, 0);
                            const long long len = (long long)v[j] - v[i];
                            const int mine = v[i] >= 0 && len > 0 && v[j] <= M;
                            bad += ec_page_seq_mine(&t, s) != mine;
                            if (mine && v[x] >= 0)
                                bad += ec_page_seq_ok(&t, s, v[x]) != (v[k] >= 0 && v[k] <= v[x] && v[k] + len <= rows);
                            seen += 2;
                        }
    printf("%ld checks, %ld wrong\n", seen, bad);
    return bad != 0;
}
