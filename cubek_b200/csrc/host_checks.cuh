// Host-side checks and launch state of api.cu that other entry-point files share.
#pragma once

#include "common.cuh"

namespace qk {

int dtype_size(int dt);
int num_quants(const QkScheme *s);
int kind_of(const QkScheme *s);
int check_scheme(const QkScheme *s);
int check_tensor(const QkTensor *t, int elem_size);
bool is_contiguous(const QkTensor *t);
bool is_row_strided(const QkTensor *t, long long *row_stride);
LaunchCfg current_cfg();
int cuda_status(cudaError_t e);
void count_launch(int n = 1);
int *stage_error_flag();  // device address of the flag a kernel raises when it gives up on a bounded wait

}  // namespace qk
