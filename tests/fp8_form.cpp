// fp8_form.cpp -- the form that a product with an epilogue takes (zz_fp8_form.h), for each line of
// standard input: packed rows, columns, rows, matrices, whether a table, whether the 8-bit instructions
// may be taken. Behind it 1 where a launch holds the call, 0 where it is declined.
#include "../zunzuncito_amd/csrc/zz_fp8_form.h"

#include <stdio.h>

int main() {
    int O, I, P, E, table, eight;
    while (scanf("%d %d %d %d %d %d", &O, &I, &P, &E, &table, &eight) == 6) 
        printf("%d %d\n", zz_f8_ep_kernel(O, I, P, E, table, eight), zz_f8_ep_fits(O, P, E, table));
    return 0;
}
