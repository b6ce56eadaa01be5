// Group normalisation with a following activation: the backward call.
#include "groupnorm_body.h"

using namespace sv;

extern "C" {

int sv_groupnorm_act_bwd(const void* x, const void* dy, const float* gamma, const float* beta, const float* save_mean,
                         const float* save_rstd, void* dx, float* dgamma, float* dbeta, int accumulate, int64_t N, int64_t S,
                         int C, int groups, int act, float alpha, void* workspace, size_t workspace_bytes, int dtype,
                         sv_stream_t stream) {
    SV_F32_OR_BF16(dtype, "sv_groupnorm_act_bwd");
    int rc = gn_check("sv_groupnorm_act_bwd", N, S, C, groups, act, workspace, workspace_bytes);
    if (rc) return rc;
    SV_REQUIRE(dgamma && dbeta, "sv_groupnorm_act_bwd: null tensor");
    hipStream_t st = to_stream(stream);
    if (N == 0) {
        hipLaunchKernelGGL(gn_param_fold_k, dim3((unsigned)ceil_div(C, 16)), dim3(1024), 0, st, nullptr, dgamma, dbeta, (int64_t)0, C,
                           accumulate);
        return check_launch("sv_groupnorm_act_bwd");
    }
    SV_REQUIRE(x && dy && gamma && beta && save_mean && save_rstd && dx, "sv_groupnorm_act_bwd: null tensor");
    GnArgs a{};
    a.x = x;
    a.dy = dy;
    a.gamma = gamma;
    a.beta = beta;
    a.mean = const_cast<float*>(save_mean);
    a.rstd = const_cast<float*>(save_rstd);
    a.out = dx;
    a.dgamma = dgamma;
    a.dbeta = dbeta;
    a.accumulate = accumulate;
    a.N = N;
    a.S = S;
    a.C = C;
    a.G = groups;
    a.D = C / groups;
    a.act = act;
    a.alpha = alpha;
    const auto run = dtype == SV_F32 ? launch<float, true> : launch<__bf16, true>;
    return run("sv_groupnorm_act_bwd", a, workspace, st);
}

}  // extern "C"
