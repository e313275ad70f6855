// int8 products grouped by expert (gnk_grouped.h).
#include "gnk_grouped.h"
GNK_DEFINE_GROUPED(gnk_grouped_i8, OP_I8, 0, 0)
