/* api_util.h -- what the files of the C host layer share: the error convention of openfish_api.c. */
#ifndef OFB_API_UTIL_H
#define OFB_API_UTIL_H

#pragma GCC visibility push(hidden)
/* Records a failure and, in the reference's error mode, ends the process. */
void ofb_api_raise(const char *func, int code, const char *text);
void ofb_api_clear(void);
/* Whether rc is a failure of the CUDA side; if so it has been raised with the CUDA side's text. */
int ofb_api_backend_failed(const char *func, int rc);
#pragma GCC visibility pop

#endif
