/* encoder.h -- the encoder's operators behind the C host layer (encoder_api.c): the arguments have been checked there.
 * Every function returns an openfish_b200_status value, its text in ofb_error_text(). */
#ifndef OFB_ENCODER_H
#define OFB_ENCODER_H

#include "openfish_b200.h"

#ifdef __cplusplus
extern "C" {
#endif
#pragma GCC visibility push(hidden)

int ofb_attention(void *stream, const openfish_b200_attention_t *a);
size_t ofb_attention_workspace(const openfish_b200_attention_t *a);
int ofb_matmul_i8(void *stream, const openfish_b200_matmul_i8_t *a);
int ofb_norm(void *stream, const openfish_b200_norm_t *a);
/* Waits for the stream; then *gave_up: whether a kernel of the file has given up a wait on this device since the calling thread's last
 * such call (before it: since its first call of the operator). */
int ofb_attention_settle(void *stream, int *gave_up);
int ofb_matmul_i8_settle(void *stream, int *gave_up);
/* The current device's count of waits that have run out. */
int ofb_attention_status(int **word);
int ofb_matmul_i8_status(int **word);

/* Leaves a text for ofb_error_text() and returns the code. */
int ofb_fail(int code, const char *text);

#pragma GCC visibility pop
#ifdef __cplusplus
}
#endif
#endif
