// Group normalisation with a following activation: the workspace and the forward call.  (The backward call is a source of its own,
// so that the two compile side by side.)
#include "groupnorm_body.h"

using namespace sv;

extern "C" {

size_t sv_groupnorm_workspace_bytes(int64_t N, int64_t S, int C, int groups) {
    if (N <= 0 || S <= 0 || C <= 0 || C > kGnMaxC || groups < 1 || C % groups) return 0;
    return gn_ws_bytes(N, S, C, groups);
}

int sv_groupnorm_form(int64_t N, int64_t S, int C, int groups, int backward, int dtype, int alignment, int32_t* form) {
    SV_F32_OR_BF16(dtype, "sv_groupnorm_form");
    SV_REQUIRE(N > 0 && S > 0 && C > 0 && C <= kGnMaxC && groups >= 1 && C % groups == 0 && form != nullptr, "sv_groupnorm_form: bad arguments");
    SV_REQUIRE(S <= ((int64_t)1 << 40) / C && N <= ((int64_t)1 << 40) / (S * C), "sv_groupnorm_form: tensor too large");
    SV_REQUIRE(alignment >= 1 && (alignment & (alignment - 1)) == 0, "sv_groupnorm_form: alignment must be a power of two");
    const GnPlan q = gn_plan(N, S, C, groups, dtype == SV_F32 ? 4 : 2, (uintptr_t)alignment, backward != 0);
    form[0] = q.K;
    form[1] = q.NT;
    form[2] = q.V;
    form[3] = q.K > 0 && q.groups;
    form[4] = q.K > 0 && q.groups && q.V * (dtype == SV_F32 ? 4 : 2) == 16 ? q.far : 0;
    form[5] = q.slabs;
    form[6] = q.K > 0 ? 1 : q.chunks;
    return SV_OK;
}

int sv_groupnorm_act_fwd(const void* x, const float* gamma, const float* beta, void* y, float* save_mean, float* save_rstd,
                         int64_t N, int64_t S, int C, int groups, float eps, int act, float alpha, void* workspace,
                         size_t workspace_bytes, int dtype, sv_stream_t stream) {
    SV_F32_OR_BF16(dtype, "sv_groupnorm_act_fwd");
    int rc = gn_check("sv_groupnorm_act_fwd", N, S, C, groups, act, workspace, workspace_bytes);
    if (rc) return rc;
    SV_REQUIRE(eps >= 0.f, "sv_groupnorm_act_fwd: epsilon must not be negative");
    SV_REQUIRE((save_mean == nullptr) == (save_rstd == nullptr), "sv_groupnorm_act_fwd: save_mean and save_rstd go together");
    if (N == 0) return SV_OK;
    SV_REQUIRE(x && gamma && beta && y, "sv_groupnorm_act_fwd: null tensor");
    GnArgs a{};
    a.x = x;
    a.gamma = gamma;
    a.beta = beta;
    a.out = y;
    a.mean = save_mean;
    a.rstd = save_rstd;
    a.N = N;
    a.S = S;
    a.C = C;
    a.G = groups;
    a.D = C / groups;
    a.eps = eps;
    a.act = act;
    a.alpha = alpha;
    const auto run = dtype == SV_F32 ? launch<float, false> : launch<__bf16, false>;
    return run("sv_groupnorm_act_fwd", a, workspace, to_stream(stream));
}

}  // extern "C"
