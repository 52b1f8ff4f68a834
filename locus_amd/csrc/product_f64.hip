// The float64 instantiations of the fused and grouped products.
#include "product_rows.h"
#include "product_tile.h"
namespace locus {
template int launch_product_tile<double>(const ProductDesc&, int, int, hipStream_t);
template int launch_product_rows<double>(const ProductDesc&, int, hipStream_t);
template bool product_pairs<double>(const ProductDesc&, int, int, const ProductDesc&, int, int);
template int launch_product_pair<double>(const ProductDesc&, int, const ProductDesc&, int, hipStream_t);
}  // namespace locus
