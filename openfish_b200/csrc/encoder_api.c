/* encoder_api.c -- the C host layer of the encoder's operators: argument checks in front of encoder.h. */
#include <limits.h>
#include <math.h>
#include <stdio.h>

#include "api_util.h"
#include "encoder.h"
#include "openfish_b200.h"

static int refuse(const char *func, int code, const char *text) {
    ofb_api_raise(func, code, text);
    return 1;
}
static int aligned(const void *p, size_t to) { return ((size_t)p & (to - 1)) == 0; }
static int bad_dtype(const char *func, int dtype) {
    if (dtype == OPENFISH_B200_F16 || dtype == OPENFISH_B200_BF16) return 0;
    return refuse(func, OPENFISH_B200_ERR_ARGUMENT, "dtype must be OPENFISH_B200_F16 or OPENFISH_B200_BF16");
}

/* A tensor [rows][heads][head_dim]: a stride counts only where there is a second element along it.  The limit on a
 * stride is that of a tensor map (40 bits of bytes). */
static int bad_heads(const char *func, const char *name, const void *p, long long rows, int heads, long long stride_row,
                     long long stride_head) {
    char msg[160];
    if (!p) {
        snprintf(msg, sizeof(msg), "%s must not be NULL", name);
        return refuse(func, OPENFISH_B200_ERR_ARGUMENT, msg);
    }
    const long long most = (1LL << 38);
    if (!aligned(p, 16) || (rows > 1 && (stride_row % 8 != 0 || stride_row < 8 || stride_row > most)) ||
        (heads > 1 && (stride_head % 8 != 0 || stride_head < 8 || stride_head > most))) {
        snprintf(msg, sizeof(msg), "%s must be 16-byte aligned, its strides positive multiples of 8", name);
        return refuse(func, OPENFISH_B200_ERR_LAYOUT, msg);
    }
    return 0;
}
/* Of a tensor that is written, the rows and heads lie next to or inside one another's gaps: no element has two places. */
static int elements_meet(long long rows, int heads, int head_dim, long long stride_row, long long stride_head) {
    if (rows < 2) return heads > 1 && stride_head < head_dim;
    if (heads < 2) return stride_row < head_dim;
    /* (the inner stride first; by division, for a product of these may pass 64 bits) */
    if (stride_head <= stride_row) return stride_head < head_dim || (stride_row - head_dim) / stride_head < heads - 1;
    return stride_row < head_dim || (stride_head - head_dim) / stride_row < rows - 1;
}

/* What does not need the pointers. */
static int bad_attention_sizes(const char *func, const openfish_b200_attention_t *a) {
    if (!a) return refuse(func, OPENFISH_B200_ERR_ARGUMENT, "args must not be NULL");
    if (bad_dtype(func, a->dtype)) return 1;
    if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8 != 0)
        return refuse(func, OPENFISH_B200_ERR_SHAPE, "head_dim must be a multiple of 8 from 8 to 128");
    if (a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads != 0)
        return refuse(func, OPENFISH_B200_ERR_SHAPE, "q_heads must be a multiple of kv_heads, both at least 1");
    if (a->sequences < 0 || a->max_q < 0 || a->max_k < 0 || a->q_rows < 0 || a->k_rows < 0)
        return refuse(func, OPENFISH_B200_ERR_SHAPE, "negative extent");
    if (a->q_rows > INT_MAX - 65536 || a->k_rows > INT_MAX - 65536 || a->max_k > INT_MAX / 4 || (double)a->max_q * a->q_heads > 1e9 ||
        ((double)a->max_q * a->q_heads / a->kv_heads / 128 + 1) * a->kv_heads * a->sequences > 1e9)
        return refuse(func, OPENFISH_B200_ERR_TOO_LONG, "more rows than the kernels count (2^31 rows, 2^29 keys and 10^9 query heads of one sequence, 10^9 tiles of 128)");
    if (!(a->scale > 0.f) || isinf(a->scale * 1.4426950408889634f)) /* (the kernels count in powers of two) */
        return refuse(func, OPENFISH_B200_ERR_ARGUMENT, "scale must be above zero and, times log2(e), finite");
    if (a->window_left < -1 || a->window_right < -1)
        return refuse(func, OPENFISH_B200_ERR_ARGUMENT, "a window is -1 (no bound) or a number of keys");
    return 0;
}
static int nothing_to_attend(const openfish_b200_attention_t *a) { return a->sequences == 0 || a->q_rows == 0 || a->max_q == 0; }

size_t openfish_b200_attention_workspace(const openfish_b200_attention_t *args) {
    ofb_api_clear();
    if (bad_attention_sizes(__func__, args) || nothing_to_attend(args)) return 0;
    return ofb_attention_workspace(args);
}

void openfish_b200_attention(void *cuda_stream, const openfish_b200_attention_t *a) {
    ofb_api_clear();
    if (bad_attention_sizes(__func__, a) || nothing_to_attend(a)) return;
    if (!a->q_start || !a->k_start) {
        refuse(__func__, OPENFISH_B200_ERR_ARGUMENT, "q_start and k_start must not be NULL");
        return;
    }
    if (!aligned(a->q_start, 4) || !aligned(a->k_start, 4) || !aligned(a->q_used, 4) || !aligned(a->k_used, 4)) {
        refuse(__func__, OPENFISH_B200_ERR_LAYOUT, "starts and used lengths must be aligned to their type");
        return;
    }
    if (bad_heads(__func__, "q", a->q, a->q_rows, a->q_heads, a->q_stride_row, a->q_stride_head) ||
        bad_heads(__func__, "out", a->out, a->q_rows, a->q_heads, a->out_stride_row, a->out_stride_head))
        return;
    if (elements_meet(a->q_rows, a->q_heads, a->head_dim, a->out_stride_row, a->out_stride_head)) {
        refuse(__func__, OPENFISH_B200_ERR_LAYOUT, "rows and heads of out must not overlap");
        return;
    }
    if (a->k_rows > 0 &&
        (bad_heads(__func__, "k", a->k, a->k_rows, a->kv_heads, a->k_stride_row, a->k_stride_head) ||
         bad_heads(__func__, "v", a->v, a->k_rows, a->kv_heads, a->v_stride_row, a->v_stride_head)))
        return;
    const size_t need = ofb_attention_workspace(a);
    if (need > 0 && (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 16))) {
        char msg[160];
        snprintf(msg, sizeof(msg), "needs a 16-byte aligned workspace of %zu bytes (openfish_b200_attention_workspace)", need);
        refuse(__func__, OPENFISH_B200_ERR_ARGUMENT, msg);
        return;
    }
    ofb_api_backend_failed(__func__, ofb_attention(cuda_stream, a));
}

static int bad_matmul_sizes(const char *func, const openfish_b200_matmul_i8_t *a) {
    if (!a) return refuse(func, OPENFISH_B200_ERR_ARGUMENT, "args must not be NULL");
    if (bad_dtype(func, a->dtype)) return 1;
    if (a->rows < 0 || a->cols < 1 || a->depth < 1)
        return refuse(func, OPENFISH_B200_ERR_SHAPE, "rows must not be negative, cols and depth at least 1");
    if (a->depth > 131071)
        return refuse(func, OPENFISH_B200_ERR_TOO_LONG, "depth above 131071: a sum could leave 32 bits");
    if (a->rows > (1LL << 30) || a->cols > (1 << 30))
        return refuse(func, OPENFISH_B200_ERR_TOO_LONG, "more than 2^30 rows or cols");
    return 0;
}

void openfish_b200_matmul_i8(void *cuda_stream, const openfish_b200_matmul_i8_t *a) {
    ofb_api_clear();
    if (bad_matmul_sizes(__func__, a) || a->rows == 0) return;
    if (!a->x || !a->w || !a->x_scale || !a->w_scale || !a->out) {
        refuse(__func__, OPENFISH_B200_ERR_ARGUMENT, "x, w, x_scale, w_scale and out must not be NULL");
        return;
    }
    if (!aligned(a->x, 16) || !aligned(a->w, 16) || (a->rows > 1 && (a->x_stride % 16 != 0 || a->x_stride < a->depth)) ||
        (a->cols > 1 && (a->w_stride % 16 != 0 || a->w_stride < a->depth))) {
        refuse(__func__, OPENFISH_B200_ERR_LAYOUT, "rows of x and w must start on 16-byte boundaries, depth or more apart");
        return;
    }
    if (!aligned(a->x_scale, 4) || !aligned(a->w_scale, 4) || !aligned(a->out, 2) || !aligned(a->bias, 2) ||
        (a->rows > 1 && a->out_stride < a->cols) || a->x_stride > (1LL << 38) || a->w_stride > (1LL << 38) || a->out_stride > (1LL << 37)) {
        refuse(__func__, OPENFISH_B200_ERR_LAYOUT, "scales, bias and out must be aligned to their types, rows of out cols or more apart");
        return;
    }
    ofb_api_backend_failed(__func__, ofb_matmul_i8(cuda_stream, a));
}

void openfish_b200_norm(void *cuda_stream, const openfish_b200_norm_t *a) {
    ofb_api_clear();
    if (!a) {
        refuse(__func__, OPENFISH_B200_ERR_ARGUMENT, "args must not be NULL");
        return;
    }
    if (bad_dtype(__func__, a->dtype)) return;
    if (a->kind < OPENFISH_B200_NORM_NONE || a->kind > OPENFISH_B200_NORM_RMS) {
        refuse(__func__, OPENFISH_B200_ERR_ARGUMENT, "kind must be NONE, LAYER or RMS");
        return;
    }
    if (a->rows < 0 || a->width < 1 || a->rows > (1LL << 30)) {
        refuse(__func__, OPENFISH_B200_ERR_SHAPE, "rows must be 0 to 2^30 and width at least 1");
        return;
    }
    if (a->width > 32768) {
        refuse(__func__, OPENFISH_B200_ERR_TOO_LONG, "width above 32768, what one block holds of a row");
        return;
    }
    if (!(a->eps >= 0.f) || isinf(a->eps)) {
        refuse(__func__, OPENFISH_B200_ERR_ARGUMENT, "eps must be finite and not negative");
        return;
    }
    if (a->kind == OPENFISH_B200_NORM_NONE && (a->weight || a->bias)) {
        refuse(__func__, OPENFISH_B200_ERR_ARGUMENT, "kind NONE takes neither weight nor bias");
        return;
    }
    if (a->rows == 0) return;
    if (!a->x || (!a->out && !a->q) || (a->q && !a->q_scale)) {
        refuse(__func__, OPENFISH_B200_ERR_ARGUMENT, "x must not be NULL, nor both out and q, nor q_scale beside q");
        return;
    }
    if (!aligned(a->x, 2) || !aligned(a->residual, 2) || !aligned(a->weight, 2) || !aligned(a->bias, 2) || !aligned(a->out, 2) ||
        !aligned(a->q_scale, 4) ||
        (a->rows > 1 && ((a->out && a->out_stride < a->width) || (a->q && a->q_stride < a->width)))) {
        refuse(__func__, OPENFISH_B200_ERR_LAYOUT, "buffers must be aligned to their types, rows of out and q width or more apart");
        return;
    }
    ofb_api_backend_failed(__func__, ofb_norm(cuda_stream, a));
}

void openfish_b200_encoder_wait(void *cuda_stream) {
    int a = 0, m = 0;
    ofb_api_clear();
    if (ofb_api_backend_failed(__func__, ofb_attention_settle(cuda_stream, &a)) ||
        ofb_api_backend_failed(__func__, ofb_matmul_i8_settle(cuda_stream, &m)))
        return;
    if (a || m) refuse(__func__, OPENFISH_B200_ERR_DEVICE_WAIT, "a kernel gave up waiting; results queued since the last such call are meaningless");
}
