// logprobs.cpp - the log probabilities' kernels on the host, of paged.cpp's program.
#include "device.hpp"

#include "token_logprobs.hip"
