// NO_CPU_VARIANT (the operators' library calls only exist in the GPU runtime)
// A transformer's feed-forward sublayer with experts out of the runtime's operators, on bfloat16:
//     sum = x + residual,  n = rms_norm(sum),  the k experts e of the largest n router^T, w their softmax,
//     y = sum + the sum over them of w_e (silu(n gate_e^T) * (n up_e^T)) down_e^T
// for `tokens` rows; how many of them each expert gets stays in GPU memory.  One generated function per size:
// expert_feed_forward_<tokens>x<hidden>x<inner>x<experts>x<k>.  And the sublayer of feed_forward.cpp with its matrices in 4 bits: four_bit_feed_forward_<tokens>x<hidden>x<inner>.
#include <tiramisu/tiramisu.h>

using namespace tiramisu;

static void generate(int tokens, int hidden, int inner, int experts, int k)
{
    const std::string name = "expert_feed_forward_" + std::to_string(tokens) + "x" + std::to_string(hidden) + "x" + std::to_string(inner) + "x" + std::to_string(experts) + "x" + std::to_string(k);
    tiramisu::init(name);

    const int places = tokens * k;
    buffer b_x("b_x", {tokens, hidden}, p_bfloat16, a_input);
    buffer b_residual("b_residual", {tokens, hidden}, p_bfloat16, a_input);
    buffer b_norm("b_norm", {hidden}, p_bfloat16, a_input);
    buffer b_router("b_router", {experts, hidden}, p_bfloat16, a_input);
    buffer b_gate("b_gate", {experts, inner, hidden}, p_bfloat16, a_input);
    buffer b_up("b_up", {experts, inner, hidden}, p_bfloat16, a_input);
    buffer b_down("b_down", {experts, hidden, inner}, p_bfloat16, a_input);
    buffer b_sum("b_sum", {tokens, hidden}, p_bfloat16, a_output);
    buffer b_y("b_y", {tokens, hidden}, p_bfloat16, a_output);
    buffer b_n("b_n", {tokens, hidden}, p_bfloat16, a_temporary);
    buffer b_logits("b_logits", {tokens, experts}, p_bfloat16, a_temporary);
    buffer b_chosen("b_chosen", {tokens, k}, p_int32, a_temporary);
    buffer b_weights("b_weights", {tokens, k}, p_float32, a_temporary);
    buffer b_offsets("b_offsets", {experts + 1}, p_int32, a_temporary);
    buffer b_rows("b_rows", {places}, p_int32, a_temporary);
    buffer b_places("b_places", {tokens, k}, p_int32, a_temporary);
    buffer b_h("b_h", {places, inner}, p_bfloat16, a_temporary);
    buffer b_out("b_out", {places, hidden}, p_bfloat16, a_temporary);
    for (buffer *b : {&b_x, &b_residual, &b_norm, &b_router, &b_gate, &b_up, &b_down, &b_sum, &b_y, &b_n, &b_logits, &b_chosen, &b_weights, &b_offsets, &b_rows, &b_places, &b_h, &b_out})
        b->tag_gpu_global();

    var once("once", 0, 1);
    computation norm({once}, hip_rms_norm(b_x, b_norm, b_n, expr(tokens), expr(hidden), 1e-6f, &b_residual, &b_sum));
    computation logits({once}, hip_linear(b_n, b_router, b_logits, expr(tokens), expr(experts), expr(hidden)));
    computation route({once}, hip_route(b_logits, b_chosen, b_weights, b_offsets, b_rows, b_places, expr(tokens), expr(experts), expr(k)));
    computation gated({once}, hip_grouped_gated_linear(b_n, b_gate, b_up, b_offsets, b_h, expr(places), expr(tokens), expr(experts), expr(inner), expr(hidden), &b_rows));
    computation down({once}, hip_grouped_linear(b_h, b_down, b_offsets, b_out, expr(places), expr(places), expr(experts), expr(hidden), expr(inner)));
    computation combined({once}, hip_combine_rows(b_out, b_places, b_y, expr(tokens), expr(k), expr(places), expr(hidden), &b_weights, &b_sum));
    norm.then(logits, computation::root).then(route, computation::root).then(gated, computation::root).then(down, computation::root).then(combined, computation::root);

    tiramisu::codegen({&b_x, &b_residual, &b_norm, &b_router, &b_gate, &b_up, &b_down, &b_sum, &b_y}, "build/" + name + ".o", true);
}

static void generate_four_bit(int tokens, int hidden, int inner)
{
    const std::string name = "four_bit_feed_forward_" + std::to_string(tokens) + "x" + std::to_string(hidden) + "x" + std::to_string(inner);
    tiramisu::init(name);

    buffer b_x("b_x", {tokens, hidden}, p_bfloat16, a_input);
    buffer b_residual("b_residual", {tokens, hidden}, p_bfloat16, a_input);
    buffer b_norm("b_norm", {hidden}, p_bfloat16, a_input);
    buffer b_gate("b_gate", {inner, (hidden + 1) / 2}, p_uint8, a_input), b_gate_scale("b_gate_scale", {inner, (hidden + 31) / 32}, p_uint8, a_input);
    buffer b_up("b_up", {inner, (hidden + 1) / 2}, p_uint8, a_input), b_up_scale("b_up_scale", {inner, (hidden + 31) / 32}, p_uint8, a_input);
    buffer b_down("b_down", {hidden, (inner + 1) / 2}, p_uint8, a_input), b_down_scale("b_down_scale", {hidden, (inner + 31) / 32}, p_uint8, a_input);
    buffer b_sum("b_sum", {tokens, hidden}, p_bfloat16, a_output);
    buffer b_y("b_y", {tokens, hidden}, p_bfloat16, a_output);
    buffer b_n("b_n", {tokens, hidden}, p_bfloat16, a_temporary);
    buffer b_h("b_h", {tokens, inner}, p_bfloat16, a_temporary);
    for (buffer *b : {&b_x, &b_residual, &b_norm, &b_gate, &b_gate_scale, &b_up, &b_up_scale, &b_down, &b_down_scale, &b_sum, &b_y, &b_n, &b_h}) b->tag_gpu_global();

    var once("once", 0, 1);
    computation norm({once}, hip_rms_norm(b_x, b_norm, b_n, expr(tokens), expr(hidden), 1e-6f, &b_residual, &b_sum));
    computation gated({once}, hip_four_bit_gated_linear(b_n, b_gate, b_up, b_gate_scale, b_up_scale, b_h, expr(tokens), expr(inner), expr(hidden)));
    computation down({once}, hip_four_bit_linear(b_h, b_down, b_down_scale, b_y, expr(tokens), expr(hidden), expr(inner), hip_activation::none, nullptr, &b_sum));
    norm.then(gated, computation::root).then(down, computation::root);

    tiramisu::codegen({&b_x, &b_residual, &b_norm, &b_gate, &b_gate_scale, &b_up, &b_up_scale, &b_down, &b_down_scale, &b_sum, &b_y}, "build/" + name + ".o", true);
}

int main(int argc, char **argv)
{
    tiramisu::backend_options_from_command_line(argc, argv);
    generate(1, 1024, 512, 32, 4);         // a token of one sequence
    generate(300, 520, 200, 6, 2);         // a ragged batch
    generate_four_bit(1, 1024, 4096);
    generate_four_bit(300, 520, 1000);
    return 0;
}
