/* C11 caller of the key-weight, eviction and linear-attention entry points: the config's layout, and what null handles answer. */
#include <stddef.h>
#include <stdio.h>
#include "psi_cuda.h"

#define FIELD(name) printf("%s %zu %zu\n", #name, offsetof(psi_linear_config, name), sizeof(((psi_linear_config*)0)->name))

int main(void) {
    const uint32_t words[2] = {0, 1};
    const float decay = 0.0f;
    float state = 0.0f;
    uint32_t kept = 0;
    int32_t status = 0;
    psi_linear* linear = NULL;
    psi_linear_config config = {1, 1, 64, 64, 1.0f, PSI_DTYPE_BF16, 1, 1, 1};
    printf("sizeof 0 %zu\n", sizeof(psi_linear_config));
    FIELD(num_k_heads);
    FIELD(num_v_heads);
    FIELD(key_dim);
    FIELD(value_dim);
    FIELD(scale);
    FIELD(dtype);
    FIELD(num_req_slots);
    FIELD(num_layers);
    FIELD(max_tokens);
    if (psi_gqa_weigh_keys(NULL, NULL, NULL, 0, &state, &state, 1) != PSI_ERR_INVALID_ARGUMENT) return 1;
    if (psi_gqa_evict(NULL, NULL, NULL, 0, words, words, words, words, 1, 0, &state, &state, 1, &kept, 1) != PSI_ERR_INVALID_ARGUMENT) return 2;
    if (psi_linear_create(NULL, &config, &linear) != PSI_ERR_INVALID_ARGUMENT) return 3;
    if (psi_linear_set_decay(NULL, 0, &decay) != PSI_ERR_INVALID_ARGUMENT) return 4;
    if (psi_linear_prepare(NULL, words, NULL, words, words, 1) != PSI_ERR_INVALID_ARGUMENT) return 5;
    if (psi_linear_attend(NULL, 0, &state, &state, &state, &state, &state) != PSI_ERR_INVALID_ARGUMENT) return 6;
    if (psi_linear_device_status(NULL, &status) != PSI_ERR_INVALID_ARGUMENT) return 7;
    if (psi_linear_destroy(NULL) != PSI_OK) return 8;
    puts("null ok");
    return 0;
}
