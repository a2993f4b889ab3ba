// Answers, a line each, which kernel a matrix product of the score head takes (opal_linear_rules.h):
//   product P TYPE M N K CUS LARGE WHOLE -> tile          weight N IN OUT TYPE -> tile splits rows
#include <cstdio>
#include <cstring>

#include "opal_linear_rules.h"

int main()
{
    char word[16];
    while (scanf("%15s", word) == 1) {
        unsigned long long a, b, c, d, e;
        int p, type, large, whole;
        if (!strcmp(word, "product")) {
            if (scanf("%d %d %llu %llu %llu %llu %d %d", &p, &type, &a, &b, &c, &d, &large, &whole) != 8) return 1;
            printf("%d\n", opal_head::product_tile(p, type, a, b, c, (int)d, large, whole));
        } else if (!strcmp(word, "weight")) {
            if (scanf("%llu %llu %llu %llu", &a, &b, &c, &e) != 4) return 1;
            const opal_head::Splits s = opal_head::weight_splits(a, (uint32_t)b, (uint32_t)c, (int)e);
            printf("%d %llu %llu\n", s.tile, (unsigned long long)s.splits, (unsigned long long)s.rows);
        } else return 1;
    }
    return 0;
}
