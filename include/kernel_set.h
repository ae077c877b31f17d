/* Umbrella header: everything the quantized-GEMM drop-in library exports, and the operators of ext/,
 * which stand beside it and have no counterpart in the reference's headers. */
#ifndef KERNEL_SET_H_
#define KERNEL_SET_H_
#include "kernel_set/types.h"
#include "kernel_set/runtime.h"
#include "kernel_set/gemm.h"
#include "kernel_set/quant.h"
#include "kernel_set/moe.h"
#include "kernel_set/activation.h"
#include "kernel_set/norm.h"
#include "kernel_set/ext/lora.h"
#include "kernel_set/ext/moe_backward.h"
#endif /* KERNEL_SET_H_ */
