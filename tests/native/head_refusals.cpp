// Calls the score head's C entry points with arguments that they must refuse, on a ctx that has no GPU behind it: every check
// happens before the first HIP call.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "opal_internal.h"

static int failures = 0;

static void want(const char *what, int rc, int code, opal_ctx *ctx, const char *word)
{
    const char *msg = opal_last_error(ctx);
    if (rc != code || !strstr(msg, word)) {
        printf("%s: got %d (%s), wanted %d with \"%s\"\n", what, rc, msg, code, word);
        failures++;
    }
}

int main()
{
    opal_ctx ctx;
    alignas(16) static float buf[64];
    float *p = buf;
    int32_t lab[4] = {1, 1, 1, 1};
    const int F = OPAL_F32, E = OPAL_EINVAL;
    char *odd = (char *)buf + 1;

    want("norm ctx", opal_layer_norm(nullptr, p, F, 4, p, p, 2, 4, 1e-5f, p, F, 4, p, p), E, nullptr, "null ctx");
    want("norm cols 0", opal_layer_norm(&ctx, p, F, 4, p, p, 2, 0, 1e-5f, p, F, 4, p, p), E, &ctx, "cols");
    want("norm cols big", opal_layer_norm(&ctx, p, F, 1u << 21, p, p, 2, (1u << 20) + 1, 1e-5f, p, F, 1u << 21, p, p), E, &ctx, "cols");
    want("norm rows", opal_layer_norm(&ctx, p, F, 4, p, p, 1ull << 31, 4, 1e-5f, p, F, 4, p, p), E, &ctx, "rows");
    want("norm eps 0", opal_layer_norm(&ctx, p, F, 4, p, p, 2, 4, 0.f, p, F, 4, p, p), E, &ctx, "eps");
    want("norm eps nan", opal_layer_norm(&ctx, p, F, 4, p, p, 2, 4, NAN, p, F, 4, p, p), E, &ctx, "eps");
    want("norm eps inf", opal_layer_norm(&ctx, p, F, 4, p, p, 2, 4, INFINITY, p, F, 4, p, p), E, &ctx, "eps");
    want("norm x", opal_layer_norm(&ctx, nullptr, F, 4, p, p, 2, 4, 1e-5f, p, F, 4, p, p), E, &ctx, "null x");
    want("norm y", opal_layer_norm(&ctx, p, F, 4, p, p, 2, 4, 1e-5f, nullptr, F, 4, p, p), E, &ctx, "null y");
    want("norm type", opal_layer_norm(&ctx, p, 3, 4, p, p, 2, 4, 1e-5f, p, F, 4, p, p), E, &ctx, "element type of x");
    want("norm ld", opal_layer_norm(&ctx, p, F, 3, p, p, 2, 4, 1e-5f, p, F, 4, p, p), E, &ctx, "row stride of x");
    want("norm ld big", opal_layer_norm(&ctx, p, F, 4, p, p, 2, 4, 1e-5f, p, F, (1u << 21) + 1, p, p), E, &ctx, "row stride of y");
    want("norm align", opal_layer_norm(&ctx, odd, F, 4, p, p, 2, 4, 1e-5f, p, F, 4, p, p), E, &ctx, "aligned");
    want("norm none", opal_layer_norm(&ctx, nullptr, F, 4, p, p, 0, 4, 1e-5f, nullptr, F, 4, p, p), 0, &ctx, "");

    const uint64_t nb = opal_layer_norm_backward_workspace(100000, 4);
    want("back stats", opal_layer_norm_backward(&ctx, p, F, 4, p, F, 4, p, nullptr, p, 100000, 4, p, F, 4, p, p, p, nb), E, &ctx, "mean");
    want("back work", opal_layer_norm_backward(&ctx, p, F, 4, p, F, 4, p, p, p, 100000, 4, p, F, 4, p, p, p, nb - 1), OPAL_ERANGE, &ctx, "workspace");
    want("back no work", opal_layer_norm_backward(&ctx, p, F, 4, p, F, 4, p, p, p, 100000, 4, p, F, 4, p, p, nullptr, nb), OPAL_ERANGE, &ctx, "workspace");
    want("back work align", opal_layer_norm_backward(&ctx, p, F, 4, p, F, 4, p, p, p, 100000, 4, p, F, 4, p, p, p + 1, nb), E, &ctx, "16-byte");
    want("back dy", opal_layer_norm_backward(&ctx, nullptr, F, 4, p, F, 4, p, p, p, 100000, 4, p, F, 4, p, p, p, nb), E, &ctx, "null dy");
    want("back dx type", opal_layer_norm_backward(&ctx, p, F, 4, p, F, 4, p, p, p, 100000, 4, p, -1, 4, p, p, p, nb), E, &ctx, "element type of dx");

    want("linear in", opal_linear(&ctx, p, 4, p, 4, F, p, 0, nullptr, 0, 0, 2, 0, 3, p, F, 3, nullptr, 0), E, &ctx, "in");
    want("linear out", opal_linear(&ctx, p, 4, p, 4, F, p, 0, nullptr, 0, 0, 2, 4, 0, p, F, 3, nullptr, 0), E, &ctx, "out");
    want("linear act", opal_linear(&ctx, p, 4, p, 4, F, p, 4, nullptr, 0, 0, 2, 4, 3, p, F, 3, nullptr, 0), E, &ctx, "activation");
    want("linear w", opal_linear(&ctx, p, 4, nullptr, 4, F, p, 0, nullptr, 0, 0, 2, 4, 3, p, F, 3, nullptr, 0), E, &ctx, "null w");
    want("linear type", opal_linear(&ctx, p, 4, p, 4, 7, p, 0, nullptr, 0, 0, 2, 4, 3, p, F, 3, nullptr, 0), E, &ctx, "element type");
    want("linear res ld", opal_linear(&ctx, p, 4, p, 4, F, p, 0, p, F, 2, 2, 4, 3, p, F, 3, nullptr, 0), E, &ctx, "residual");
    want("linear pre ld", opal_linear(&ctx, p, 4, p, 4, F, p, 0, nullptr, 0, 0, 2, 4, 3, p, F, 3, p, 2), E, &ctx, "pre");
    want("grad_input pre", opal_linear_grad_input(&ctx, p, 3, p, 4, F, nullptr, 0, 1, nullptr, 0, 0, 2, 4, 3, p, F, 4), E, &ctx, "pre-activation");
    want("grad_input dx", opal_linear_grad_input(&ctx, p, 3, p, 4, F, nullptr, 0, 0, nullptr, 0, 0, 2, 4, 3, nullptr, F, 4), E, &ctx, "null dx");

    const uint64_t nw = opal_linear_grad_weight_workspace(2, 4, 3, F);
    const uint64_t many = opal_linear_grad_weight_workspace(100000, 4, 3, F);
    want("grad_weight work", opal_linear_grad_weight(&ctx, p, 3, p, 4, F, 100000, 4, 3, p, 4, p, p, many - 1), OPAL_ERANGE, &ctx, "workspace");
    want("grad_weight no work", opal_linear_grad_weight(&ctx, p, 3, p, 4, F, 100000, 4, 3, p, 4, p, nullptr, many), OPAL_ERANGE, &ctx, "workspace");
    want("grad_weight dw", opal_linear_grad_weight(&ctx, p, 3, p, 4, F, 2, 4, 3, nullptr, 4, nullptr, p, nw), E, &ctx, "null dw");
    want("grad_weight dw ld", opal_linear_grad_weight(&ctx, p, 3, p, 4, F, 2, 4, 3, p, 3, p, p, nw), E, &ctx, "row stride of dw");
    want("grad_weight dy", opal_linear_grad_weight(&ctx, nullptr, 3, p, 4, F, 2, 4, 3, p, 4, p, p, nw), E, &ctx, "null dy");
    want("grad_weight type", opal_linear_grad_weight(&ctx, nullptr, 3, nullptr, 4, 5, 0, 4, 3, p, 4, p, p, nw), E, &ctx, "element type");

    want("loss labels", opal_softmax_loss(&ctx, p, F, 4, 2, 4, nullptr, 1.f, p, p, F, 4), E, &ctx, "labels");
    want("loss nothing", opal_softmax_loss(&ctx, p, F, 4, 2, 4, lab, 1.f, nullptr, nullptr, F, 4), E, &ctx, "neither");
    want("loss grad ld", opal_softmax_loss(&ctx, p, F, 4, 2, 4, lab, 1.f, p, p, F, 3), E, &ctx, "row stride of grad");
    want("loss K", opal_softmax_loss(&ctx, p, F, 4, 2, 0, lab, 1.f, p, p, F, 3), E, &ctx, "K");
    want("class out", opal_softmax_class(&ctx, p, F, 4, 2, 4, nullptr, p), E, &ctx, "d_out_class");
    want("class ctx", opal_softmax_class(nullptr, p, F, 4, 2, 4, lab, p), E, nullptr, "null ctx");

    // an output over an input: with another type or row stride, or where no input may be overwritten
    const int H = OPAL_BF16;
    float *q = buf + 32;
    want("norm over x", opal_layer_norm(&ctx, p, F, 4, nullptr, nullptr, 2, 4, 1e-5f, p, H, 4, nullptr, nullptr), E, &ctx, "same place");
    want("norm over x ld", opal_layer_norm(&ctx, p, F, 4, nullptr, nullptr, 2, 4, 1e-5f, p, F, 5, nullptr, nullptr), E, &ctx, "same place");
    want("back over x", opal_layer_norm_backward(&ctx, q, F, 4, p, F, 4, p, p, p, 100000, 4, p, F, 8, p, p, p, nb), E, &ctx, "same place");
    want("back over dy", opal_layer_norm_backward(&ctx, q, F, 4, p, F, 4, p, p, p, 100000, 4, q, H, 4, p, p, p, nb), E, &ctx, "same place");
    want("linear over res", opal_linear(&ctx, p, 4, p + 8, 4, F, nullptr, 0, q, F, 4, 2, 4, 3, q, F, 3, nullptr, 0), E, &ctx, "same place");
    want("linear over x", opal_linear(&ctx, p, 4, p + 8, 4, F, nullptr, 0, nullptr, 0, 0, 2, 4, 3, p, F, 3, nullptr, 0), E, &ctx, "own");
    want("linear over w", opal_linear(&ctx, p, 4, p + 8, 4, F, nullptr, 0, nullptr, 0, 0, 2, 4, 3, p + 8, F, 3, nullptr, 0), E, &ctx, "own");
    want("linear pre over y", opal_linear(&ctx, p, 4, p + 8, 4, F, nullptr, 0, nullptr, 0, 0, 2, 4, 3, q, F, 3, q, 3), E, &ctx, "own");
    want("grad_input over dy", opal_linear_grad_input(&ctx, p, 3, q, 4, F, nullptr, 0, 0, nullptr, 0, 0, 2, 4, 3, p, F, 4), E, &ctx, "own");
    want("grad_input over res", opal_linear_grad_input(&ctx, p, 3, p + 8, 4, F, nullptr, 0, 0, q, F, 4, 2, 4, 3, q, H, 4), E, &ctx, "same place");
    want("loss over scores", opal_softmax_loss(&ctx, p, F, 4, 2, 4, lab, 1.f, q, p, H, 4), E, &ctx, "same place");

    // sizes that the calls refuse need no workspace
    const uint32_t none = 0, big = (1u << 20) + 1;
    if (opal_linear_grad_weight_workspace(100, none, 3, F) || opal_linear_grad_weight_workspace(100, 3, none, F) || opal_linear_grad_weight_workspace(100, big, 3, F) ||
        opal_linear_grad_weight_workspace(100, 3, big, H) || opal_linear_grad_weight_workspace(~0ull, 3, 3, F) || opal_layer_norm_backward_workspace(100, none) ||
        opal_layer_norm_backward_workspace(100, big) || opal_layer_norm_backward_workspace(~0ull, 4)) {
        printf("a workspace for sizes that are refused\n");
        failures++;
    }
    if (failures) return 1;
    printf("head refusals: ok\n");
    return 0;
}
