// NO_CPU_VARIANT (the operators' library calls only exist in the GPU runtime)
// A transformer's feed-forward sublayer out of the runtime's operators, on bfloat16:
//     sum = x + residual,  n = rms_norm(sum),  h = silu(n gate^T) * (n up^T),  y = sum + h down^T
// for `tokens` rows: the residual stream's addition and norm, both projections of the gated layer in one kernel, and the down projection with the
// residual's addition in its epilogue.  One generated function per size: feed_forward_<tokens>x<hidden>x<inner>.
#include <tiramisu/tiramisu.h>

using namespace tiramisu;

static void generate(int tokens, int hidden, int inner)
{
    const std::string name = "feed_forward_" + std::to_string(tokens) + "x" + std::to_string(hidden) + "x" + std::to_string(inner);
    tiramisu::init(name);

    buffer b_x("b_x", {tokens, hidden}, p_bfloat16, a_input);
    buffer b_residual("b_residual", {tokens, hidden}, p_bfloat16, a_input);
    buffer b_norm("b_norm", {hidden}, p_bfloat16, a_input);
    buffer b_gate("b_gate", {inner, hidden}, p_bfloat16, a_input);
    buffer b_up("b_up", {inner, hidden}, p_bfloat16, a_input);
    buffer b_down("b_down", {hidden, inner}, p_bfloat16, a_input);
    buffer b_sum("b_sum", {tokens, hidden}, p_bfloat16, a_output);
    buffer b_y("b_y", {tokens, hidden}, p_bfloat16, a_output);
    buffer b_n("b_n", {tokens, hidden}, p_bfloat16, a_temporary);
    buffer b_h("b_h", {tokens, inner}, p_bfloat16, a_temporary);
    for (buffer *b : {&b_x, &b_residual, &b_norm, &b_gate, &b_up, &b_down, &b_sum, &b_y, &b_n, &b_h}) b->tag_gpu_global();

    computation norm({var("once", 0, 1)}, hip_rms_norm(b_x, b_norm, b_n, expr(tokens), expr(hidden), 1e-6f, &b_residual, &b_sum));
    computation gated({var("once", 0, 1)}, hip_gated_linear(b_n, b_gate, b_up, b_h, expr(tokens), expr(inner), expr(hidden)));
    computation down({var("once", 0, 1)}, hip_linear(b_h, b_down, b_y, expr(tokens), expr(hidden), expr(inner), hip_activation::none, nullptr, &b_sum));
    norm.then(gated, computation::root).then(down, computation::root);

    tiramisu::codegen({&b_x, &b_residual, &b_norm, &b_gate, &b_up, &b_down, &b_sum, &b_y}, "build/" + name + ".o", true);
}

int main(int argc, char **argv)
{
    tiramisu::backend_options_from_command_line(argc, argv);
    generate(1, 1024, 4096);       // a token of one sequence
    generate(300, 520, 1000);      // a ragged batch
    generate(2048, 1024, 4096);    // a prompt
    return 0;
}
