// The rules of csrc/host/block8_plan.cpp over sizes of all kinds: what they give is what the kernels take, and each variant is some call's.
#include "../alphasparse_b200/csrc/host/block8_plan.cpp"

#include <stdio.h>
#include <stdlib.h>

#include <set>
#include <utility>

using namespace asp::host;

#define CHECK(c)                                           \
    do                                                     \
    {                                                      \
        if (!(c))                                          \
        {                                                  \
            printf("line %d: %s\n", __LINE__, #c);         \
            return 1;                                      \
        }                                                  \
    } while (0)

int main()
{
    const int sms = 148;
    // clusters that run at once on a chip whose parts have 18 SMs, two CTAs an SM and one
    unsigned fit2[9] = {}, fit1[9] = {};
    for (unsigned s = 1; s <= 8; s++) fit2[s] = 8 * (36 / s) + (s <= 8 ? 8 / s : 0), fit1[s] = 8 * (18 / s) + (s <= 4 ? 4 / s : 0);
    std::set<unsigned> few, batch;
    std::set<bool> which;
    std::set<std::pair<unsigned, unsigned>> products, gradients;
    for (unsigned rows = 1; rows < 70000; rows = rows < 160 ? rows + 1 : rows * 3 / 2)
        for (unsigned longest = 0; longest < 3000; longest = longest * 2 + 1)
        {
            const unsigned s = block8_few_split(rows, longest, 1, fit2);
            for (unsigned per : {2u, 4u}) CHECK(block8_few_split(rows, longest, per, fit2) == (longest <= per ? 1 : s));
            CHECK(s >= 1 && s <= 8 && (s == 1 || s <= longest) && (s == 1 || rows <= fit2[s]));
            few.insert(s);
            const unsigned b = block8_batch_split(rows, longest, sms, fit2);
            CHECK(b >= 1 && b <= s && (b == s || rows * b <= (unsigned)sms));
            batch.insert(b);
            for (unsigned n : {1u, 8u, 9u, 32u}) which.insert(block8_batch(rows, longest, n, false, sms, fit2));
            CHECK(!block8_batch(rows, longest, 32, true, sms, fit2) || (block8_batch(rows, longest, 32, false, sms, fit2) && longest <= b * kBlock8Sum));
            for (unsigned n = 33; n < 100000; n = n * 3 / 2)
            {
                const Block8ProductPlan p = block8_product_plan(rows, (unsigned)(0.7 * rows * longest), longest, n, sms, fit1);
                CHECK(p.tile % 64 == 0 && p.tile >= 64 && p.tile <= kBlock8ProductRows && p.split >= 1 && p.split <= 8);
                // a CTA of a cluster has one tile, and all of them run at once
                CHECK(p.split == 1 || ((unsigned long long)rows * ((n + p.tile - 1) / p.tile) <= fit1[p.split] && longest >= 2 * p.split));
                products.insert({p.tile, p.split});
            }
        }
    for (unsigned columns = 1; columns < 3000; columns = columns * 3 / 2 + 1)
        for (unsigned each = 1; each <= 40; each++)
        {
            for (unsigned n = 1; n < 100000; n = n * 2 + 1)
            {
                const Block8GradientPlan p = block8_gradient_plan(columns * each, columns * (each / 2), n, sms, fit1);
                CHECK((p.most == 1 || (p.most == 2 && each > 1)) && (p.split == 1 || p.split == 2 || p.split == 4 || p.split == 8));
                CHECK(p.split <= (n + kBlock8GradientRows - 1) / kBlock8GradientRows); // each CTA has a step, so that its sums are there
                CHECK(p.split == 1 || (p.most == 1 && columns * each <= fit1[p.split]));
                gradients.insert({p.most, p.split});
            }
        }
    for (unsigned s = 1; s <= 8; s++) CHECK(few.count(s) && batch.count(s));
    CHECK(which.size() == 2);
    for (unsigned t : {64u, 128u, 192u}) CHECK(products.count({t, 1}));
    for (unsigned s : {2u, 4u, 8u}) CHECK(products.count({64, s}));
    for (unsigned s : {1u, 2u, 4u, 8u}) CHECK(gradients.count({1, s}));
    CHECK(gradients.count({2, 1}));
    printf("%zu, %zu, %zu variants\n", few.size(), products.size(), gradients.size());
    return 0;
}
