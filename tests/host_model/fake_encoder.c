/* The host layer of the encoder's operators over a CUDA side made for the purpose: calls that fail when told to, kernels that
 * have given up when told to, and a count of what was called.  Test code only. */
#include "../../openfish_b200/csrc/encoder.h"

#pragma GCC visibility push(default)
int fake_fails = 0, fake_gave_up[2] = {0, 0}, fake_calls = 0;
size_t fake_workspace = 0;
#pragma GCC visibility pop

static int answer(void) {
    ++fake_calls;
    return fake_fails ? OPENFISH_B200_ERR_CUDA : OPENFISH_B200_OK;
}
int ofb_attention(void *stream, const openfish_b200_attention_t *a) { return answer(); }
size_t ofb_attention_workspace(const openfish_b200_attention_t *a) { return fake_workspace; }
int ofb_matmul_i8(void *stream, const openfish_b200_matmul_i8_t *a) { return answer(); }
int ofb_norm(void *stream, const openfish_b200_norm_t *a) { return answer(); }
int ofb_attention_settle(void *stream, int *gave_up) {
    *gave_up = fake_gave_up[0];
    return answer();
}
int ofb_matmul_i8_settle(void *stream, int *gave_up) {
    *gave_up = fake_gave_up[1];
    return answer();
}
