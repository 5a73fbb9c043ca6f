/* A C99 consumer of include/ncz_paged.h, built and run by tests/test_paged.py
 * on the CPU: fills every descriptor and checks that bad calls are refused
 * before any device is touched.  Exit status 0 = every check passed. */
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "ncz_flash.h"
#include "ncz_paged.h"

#define CHECK(cond)                                                      \
    do {                                                                 \
        if (!(cond)) {                                                   \
            fprintf(stderr, "check failed at line %d: %s\n", __LINE__, #cond); \
            return 1;                                                    \
        }                                                                \
    } while (0)

int main(void) {
    ncz_paged_cache c;
    ncz_paged_plan_desc plan;
    ncz_paged_append_desc append;
    ncz_paged_decode_desc decode;
    size_t bytes = 0;

    memset(&c, 0, sizeof c);
    c.k = (void *)(uintptr_t)0x10000000u;
    c.v = (void *)(uintptr_t)0x20000000u;
    c.num_pages = 100;
    c.page_size = 16;
    c.kv_heads = 8;
    c.head_dim = 128;
    c.k_head_stride = c.v_head_stride = 128;
    c.k_token_stride = c.v_token_stride = 8 * 128;
    c.k_page_stride = c.v_page_stride = 16 * 8 * 128;
    c.dtype = NCZ_DTYPE_E4M3;
    CHECK(ncz_paged_validate(&c) == NCZ_SUCCESS);
    CHECK(ncz_paged_validate(NULL) == NCZ_ERROR_INVALID_VALUE);
    CHECK(ncz_paged_decode_workspace(&c, 12, -1, &bytes) == NCZ_ERROR_INVALID_VALUE);

    memset(&plan, 0, sizeof plan);
    plan.device = -1;
    CHECK(ncz_paged_plan(&plan) == NCZ_ERROR_INVALID_VALUE);
    CHECK(ncz_paged_plan(NULL) == NCZ_ERROR_INVALID_VALUE);

    memset(&append, 0, sizeof append);
    append.device = -1;
    append.in_dtype = NCZ_DTYPE_BF16;
    CHECK(ncz_paged_append(&c, &append) == NCZ_SUCCESS); /* no tokens: nothing to do */
    append.tokens = 1;
    CHECK(ncz_paged_append(&c, &append) == NCZ_ERROR_INVALID_VALUE);

    memset(&decode, 0, sizeof decode);
    decode.device = -1;
    decode.q_heads = 32;
    decode.q_dtype = decode.o_dtype = NCZ_DTYPE_BF16;
    CHECK(ncz_paged_decode(&c, &decode) == NCZ_SUCCESS); /* an empty batch */
    decode.batch = 1;
    CHECK(ncz_paged_decode(&c, &decode) == NCZ_ERROR_INVALID_VALUE);
    c.v_head_stride = 64; /* rows overlap */
    CHECK(ncz_paged_decode(&c, &decode) == NCZ_ERROR_INVALID_VALUE);

    printf("paged consumer: ok\n");
    return 0;
}
