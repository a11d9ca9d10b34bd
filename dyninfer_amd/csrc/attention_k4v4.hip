// Attention over K codes of 4 bits and V codes of 4 bits.
#include "attention_impl.hpp"

DMX_ATTEND_INSTANCE(4, 4)
