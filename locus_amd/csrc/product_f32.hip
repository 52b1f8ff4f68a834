// The float32 instantiations of the fused and grouped products.
#include "product_rows.h"
#include "product_tile.h"
namespace locus {
template int launch_product_tile<float>(const ProductDesc&, int, int, hipStream_t);
template int launch_product_rows<float>(const ProductDesc&, int, hipStream_t);
template bool product_pairs<float>(const ProductDesc&, int, int, const ProductDesc&, int, int);
template int launch_product_pair<float>(const ProductDesc&, int, const ProductDesc&, int, hipStream_t);
}  // namespace locus
