// The rules of psh_linear_plan.h for a descriptor, as a function that tests load.
#include "psh_linear_plan.h"

// kinds of tiles of: the forward call, the gradient of x, that of the weights; whether the latter two are one launch; rows of a piece; bytes of scratch memory
extern "C" void plan(const psh_linear_desc* d, int64_t* out) {
    const GradPlan p = grad_plan(d);
    out[0] = forward_kind(d);
    out[1] = p.rows;
    out[2] = p.weights;
    out[3] = p.joint;
    out[4] = grad_piece(d, grad_direct(d));
    out[5] = grad_space(d).total;
}
