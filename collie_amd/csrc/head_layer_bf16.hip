#include "head_layer_impl.h"

template struct collie::HeadLayer<collie::bf16_t>;
