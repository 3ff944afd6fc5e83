#include "head_layer_impl.h"

template struct collie::HeadLayer<float>;
