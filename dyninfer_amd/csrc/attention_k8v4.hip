// Attention over K codes of 8 bits and V codes of 4 bits.
#include "attention_impl.hpp"

DMX_ATTEND_INSTANCE(8, 4)
