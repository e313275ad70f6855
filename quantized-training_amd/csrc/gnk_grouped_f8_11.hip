// fp8 products grouped by expert (gnk_grouped.h): A e5m2, B e5m2.
#include "gnk_grouped.h"
GNK_DEFINE_GROUPED(gnk_grouped_f8_11, OP_F8, 1, 1)
