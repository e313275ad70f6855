// fp8 products grouped by expert (gnk_grouped.h): A e5m2, B e4m3.
#include "gnk_grouped.h"
GNK_DEFINE_GROUPED(gnk_grouped_f8_10, OP_F8, 1, 0)
