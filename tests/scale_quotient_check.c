/* hn_common.cuh: quot_const with 127 (the int8 scale absmax / 127) against the IEEE quotient, for every positive finite fp32
 * absmax: K that is normed and rotated in fp32 is scaled from such peaks, not only from bf16 ones. */
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

static float quot_const(float p, float d, float rd) {
    const volatile float q0 = p * rd;       /* rounded to fp32 here */
    return fmaf(fmaf(-q0, d, p), rd, q0);
}

int main(void) {
    long long bad = 0, n = 0;
#pragma omp parallel for reduction(+ : bad, n) schedule(static)
    for (int64_t u = 1; u < 0x7f800000LL; ++u) {
        const uint32_t bits = (uint32_t)u;
        float p;
        memcpy(&p, &bits, 4);
        bad += quot_const(p, 127.0f, 1.0f / 127.0f) != p / 127.0f;
        ++n;
    }
    printf("%lld values, mismatches %lld\n", n, bad);
    return bad != 0;
}
