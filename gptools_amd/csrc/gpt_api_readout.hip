// Read-out of several latent fields (include/gptools_hip.h): argument checks of the layer norm and of the categorical log
// density. The kernels take all memory from the caller, so these calls are safe in a captured graph from the first one on.
#include "gpt_ctx.h"
#include "gpt_readout.h"
using namespace gptd;

namespace {

// the context's device for the time of a call
struct OnDevice {
    int before = -1;
    hipError_t err;
    explicit OnDevice(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else before = -1;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

__global__ __launch_bounds__(256) void fill_zero(unsigned char* p, size_t bytes) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < bytes; i += (size_t)gridDim.x * 256) p[i] = 0;
}
int zero(gpt_ctx* c, void* p, size_t bytes) {
    if (!p || !bytes) return GPT_OK;
    const size_t blocks = (bytes + 255) / 256;
    fill_zero<<<dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, c->stream>>>((unsigned char*)p, bytes);
    HIP_TRY(c, hipGetLastError());
    return GPT_OK;
}

bool known_type(int dtype) { return dtype == GPT_F64 || dtype == GPT_F32 || dtype == GPT_F16 || dtype == GPT_BF16; }
size_t size_of(int dtype) { return dtype == GPT_F64 ? 8 : dtype == GPT_F32 ? 4 : 2; }
constexpr int64_t MOST = 2147483647LL;                                       // rows
constexpr int64_t MOST_FEATURES = (int64_t)1 << 21, MOST_CLASSES = (int64_t)1 << 26;
constexpr int64_t MOST_WIDTH = (int64_t)1 << 40;

int check_norm(gpt_ctx* c, int dtype, int64_t rows, int64_t width) {
    if (!known_type(dtype)) return fail(c, GPT_ERR_UNSUPPORTED, "unknown element type");
    if (rows < 0 || width < 1) return fail(c, GPT_ERR_SHAPE, "layer norm needs rows >= 0 and width >= 1");
    if (rows > MOST || width > MOST_WIDTH) return fail(c, GPT_ERR_SHAPE, "layer norm: too many rows, or rows too long");
    return GPT_OK;
}
int check_class(gpt_ctx* c, int dtype, int64_t ldx, int64_t ldbeta, int64_t rows, int64_t features, int64_t classes) {
    if (!known_type(dtype)) return fail(c, GPT_ERR_UNSUPPORTED, "unknown element type");
    if (rows < 0 || features < 1 || classes < 1)
        return fail(c, GPT_ERR_SHAPE, "categorical_logit_glm needs rows >= 0, features >= 1 and classes >= 1");
    if (rows > MOST || features > MOST_FEATURES || classes > MOST_CLASSES)
        return fail(c, GPT_ERR_SHAPE, "categorical_logit_glm: too many rows, features or classes");
    if (ldx < features || ldbeta < features) return fail(c, GPT_ERR_SHAPE, "rows of x and beta must not overlap (ldx, ldbeta >= features)");
    return GPT_OK;
}
int check_space(gpt_ctx* c, const void* ws, size_t have, size_t need) {
    if (need && (!ws || have < need)) return fail(c, GPT_ERR_SHAPE, "the workspace is too small");
    if ((uintptr_t)ws & 255) return fail(c, GPT_ERR_SHAPE, "the workspace must be 256-byte aligned");
    return GPT_OK;
}

int run_class(gpt_ctx* c, int dtype, const ClassArgs& a, bool vjp, size_t have) {
    int rc = check_class(c, dtype, a.ldx, a.ldbeta, a.rows, a.features, a.classes);
    if (rc) return rc;
    const OnDevice on(c->device);
    HIP_TRY(c, on.err);
    if (a.rows == 0) {
        if (!vjp) return GPT_OK;
        if ((rc = zero(c, a.alphabar, size_of(dtype) * (size_t)a.classes)) != GPT_OK) return rc;
        return zero(c, a.betabar, size_of(dtype) * (size_t)(a.classes * a.features));
    }
    if (!a.y || !a.x || !a.beta || !a.lp) return fail(c, GPT_ERR_SHAPE, "y, x, beta and lp must not be null");
    if (vjp && (!a.xbar || !a.betabar)) return fail(c, GPT_ERR_SHAPE, "xbar and betabar must not be null");
    if ((rc = check_space(c, a.ws, have, gpt_class_workspace(dtype, a.rows, a.features, a.classes, vjp))) != GPT_OK) return rc;
    HIP_TRY(c, gpt_launch_class(dtype, a, vjp, c->stream));
    return GPT_OK;
}

} // namespace

extern "C" {

size_t gpt_layer_norm_workspace(int dtype, int64_t rows, int64_t width, int vjp) {
    return known_type(dtype) && rows > 0 && rows <= MOST && width > 0 && width <= MOST_WIDTH ? gpt_norm_workspace(dtype, rows, width, vjp != 0) : 0;
}

int gpt_layer_norm(gpt_ctx* c, int dtype, const void* x, const void* weight, const void* bias, int64_t rows, int64_t width,
                   double eps, void* y, void* mean, void* rstd, void* workspace, size_t workspace_bytes) {
    if (!c) return GPT_ERR_SHAPE;
    int rc = check_norm(c, dtype, rows, width);
    if (rc) return rc;
    if (!(eps >= 0.0 && eps < INFINITY)) return fail(c, GPT_ERR_SHAPE, "eps must be non-negative and finite");
    if (rows == 0) return GPT_OK;
    if (!x || !y || !mean || !rstd) return fail(c, GPT_ERR_SHAPE, "x, y, mean and rstd must not be null");
    if ((rc = check_space(c, workspace, workspace_bytes, gpt_norm_workspace(dtype, rows, width, false))) != GPT_OK) return rc;
    const OnDevice on(c->device);
    HIP_TRY(c, on.err);
    NormArgs a = {};
    a.x = x;
    a.weight = weight;
    a.bias = bias;
    a.y = y;
    a.mean = mean;
    a.rstd = rstd;
    a.partial = workspace;
    a.rows = rows;
    a.width = width;
    a.eps = eps;
    HIP_TRY(c, gpt_launch_norm(dtype, a, c->stream));
    return GPT_OK;
}

int gpt_layer_norm_vjp(gpt_ctx* c, int dtype, const void* x, const void* weight, const void* mean, const void* rstd,
                       const void* ybar, int64_t rows, int64_t width, void* xbar, void* wbar, void* bbar, void* workspace,
                       size_t workspace_bytes) {
    if (!c) return GPT_ERR_SHAPE;
    int rc = check_norm(c, dtype, rows, width);
    if (rc) return rc;
    if (!wbar != !bbar) return fail(c, GPT_ERR_SHAPE, "wbar and bbar: both or neither");
    const OnDevice on(c->device);
    HIP_TRY(c, on.err);
    if (rows == 0) {
        if ((rc = zero(c, wbar, size_of(dtype) * (size_t)width)) != GPT_OK) return rc;
        return zero(c, bbar, size_of(dtype) * (size_t)width);
    }
    if (!x || !mean || !rstd || !ybar || !xbar) return fail(c, GPT_ERR_SHAPE, "x, mean, rstd, ybar and xbar must not be null");
    if ((rc = check_space(c, workspace, workspace_bytes, gpt_norm_workspace(dtype, rows, width, true))) != GPT_OK) return rc;
    NormArgs a = {};
    a.x = x;
    a.weight = weight;
    a.mean = const_cast<void*>(mean);
    a.rstd = const_cast<void*>(rstd);
    a.ybar = ybar;
    a.xbar = xbar;
    a.wbar = wbar;
    a.bbar = bbar;
    a.partial = workspace;
    a.rows = rows;
    a.width = width;
    HIP_TRY(c, gpt_launch_norm_vjp(dtype, a, c->stream));
    return GPT_OK;
}

size_t gpt_categorical_logit_glm_workspace(int dtype, int64_t rows, int64_t features, int64_t classes, int vjp) {
    return known_type(dtype) && rows > 0 && features > 0 && classes > 0 && rows <= MOST && features <= MOST_FEATURES && classes <= MOST_CLASSES
               ? gpt_class_workspace(dtype, rows, features, classes, vjp != 0)
               : 0;
}

int gpt_categorical_logit_glm_lpmf(gpt_ctx* c, int dtype, const int64_t* y, const void* x, int64_t ldx, const void* alpha,
                                   const void* beta, int64_t ldbeta, int64_t rows, int64_t features, int64_t classes, void* lp,
                                   void* workspace, size_t workspace_bytes) {
    if (!c) return GPT_ERR_SHAPE;
    ClassArgs a = {};
    a.y = y;
    a.x = x;
    a.ldx = ldx;
    a.alpha = alpha;
    a.beta = beta;
    a.ldbeta = ldbeta;
    a.rows = rows;
    a.features = features;
    a.classes = classes;
    a.lp = lp;
    a.ws = workspace;
    return run_class(c, dtype, a, false, workspace_bytes);
}

int gpt_categorical_logit_glm_lpmf_vjp(gpt_ctx* c, int dtype, const int64_t* y, const void* x, int64_t ldx, const void* alpha,
                                       const void* beta, int64_t ldbeta, const void* lpbar, int64_t rows, int64_t features,
                                       int64_t classes, void* lp, void* xbar, void* alphabar, void* betabar, void* workspace,
                                       size_t workspace_bytes) {
    if (!c) return GPT_ERR_SHAPE;
    ClassArgs a = {};
    a.y = y;
    a.x = x;
    a.ldx = ldx;
    a.alpha = alpha;
    a.beta = beta;
    a.ldbeta = ldbeta;
    a.lpbar = lpbar;
    a.rows = rows;
    a.features = features;
    a.classes = classes;
    a.lp = lp;
    a.xbar = xbar;
    a.alphabar = alphabar;
    a.betabar = betabar;
    a.ws = workspace;
    return run_class(c, dtype, a, true, workspace_bytes);
}

} // extern "C"
