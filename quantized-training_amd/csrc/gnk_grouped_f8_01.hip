// fp8 products grouped by expert (gnk_grouped.h): A e4m3, B e5m2.
#include "gnk_grouped.h"
GNK_DEFINE_GROUPED(gnk_grouped_f8_01, OP_F8, 0, 1)
