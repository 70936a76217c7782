// Entry points of the dropout kernel (dropout.cu), as torch_tokens.cpp and ops/dropout.py call them.
#pragma once

#ifdef __cplusplus
extern "C" {
#endif
int ccf_dropout(const void* x, const void* residual, void* y, const long long* state, long long* state_copy, unsigned int call,
                unsigned int drop, long long n, int type, void* stream);
#ifdef __cplusplus
}
#endif
