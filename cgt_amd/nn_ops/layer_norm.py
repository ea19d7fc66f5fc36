"""Layer norm ops: the normalisation over the last axis, and the same behind a dropout and a residual add.

The reference has no counterpart; they stand beside its cross-channel LRN ops (cgt/nn_ops/cross_channel_lrn.py)
and follow their shape: a tuple-valued forward op that keeps what the gradient needs.
"""
import ctypes

from .. import core


def _check_operands(name, input_types, weights, same):
    x = input_types[0]
    assert all(t.dtype == "f4" for t in [x] + [input_types[i] for i in weights + same]), "%s takes float32 arrays" % name
    assert x.ndim >= 1, "%s takes arrays of at least one axis" % name
    assert all(input_types[i].ndim == 1 for i in weights), "%s takes weights of one axis" % name
    assert all(input_types[i].ndim == x.ndim for i in same), "%s: operands of different ranks" % name


def _check_shapes(name, x, weights, same):
    xs = core.shape(x)
    if xs[-1] == 0 and all(n != 0 for n in xs[:-1]):
        raise ValueError("%s: rows of no columns have no statistics (shape %s)" % (name, xs))
    for w in weights:
        if core.shape(w) != xs[-1:]:
            raise ValueError("%s: weights of shape %s do not fit rows of %d columns" % (name, core.shape(w), xs[-1]))
    for s in same:
        if core.shape(s) != xs:
            raise ValueError("%s: mismatched shapes %s %s" % (name, xs, core.shape(s)))


# what every closure below starts with: the rows and columns of x, and that the weights fit them
_ROWS = r"""
                long cols = X->shape()[X->ndim() - 1], rows = cols ? X->size() / cols : 0;
"""


class LayerNorm(core.Op):
    """inputs [x, gamma, beta] -> (y, mean, rstd), the statistics with the shape of x's other axes."""
    available_impls = ("native_gpu",)

    def __init__(self, eps):
        self.eps = float(eps)

    def typ_apply(self, input_types):
        _check_operands("LayerNorm", input_types, [1, 2], [])
        stat = core.TensorType("f4", input_types[0].ndim - 1)
        return core.TupleType(input_types[0], stat, stat)

    def shp_apply(self, inputs):
        _check_shapes("LayerNorm", inputs[0], inputs[1:3], [])
        s = core.shape(inputs[0])
        return (s, s[:-1], s[:-1])

    def pullback(self, inputs, output, gout):
        x, gamma, _beta = inputs
        _y, mean, rstd = core.unpack(output)
        if any(g is not None for g in gout[1:]):
            raise core.MethodNotDefined("LayerNorm: gradients go through y only, not through the statistics")
        return core.unpack(core.Result(LayerNormBackward(), [x, gamma, mean, rstd, gout[0]]))

    def get_native_compile_info(self, input_types, devtype):
        assert devtype == "gpu"
        code = r"""
            CGT_EXPORT_C void $function($closure* cl, cgtArray** reads, cgtTuple* write) {
                cgtArray *X = reads[0], *gamma = reads[1], *beta = reads[2];
                cgtArray *y = (cgtArray*)write->getitem(0), *mean = (cgtArray*)write->getitem(1), *rstd = (cgtArray*)write->getitem(2);
""" + _ROWS + r"""
                cgt_check(gamma->size() == cols && beta->size() == cols && y->size() == X->size() && mean->size() == rows && rstd->size() == rows,
                          "LayerNorm: weights or outputs do not fit the input");
                if (cgtGlobalStatus != cgtStatusOK) return;
                int rc = cgt_amd_layer_norm_fwd_f32((const float*)X->data(), rows, cols, (const float*)gamma->data(), (const float*)beta->data(),
                    cl->eps, (float*)y->data(), (float*)mean->data(), (float*)rstd->data(), cgt_get_stream());
                cgt_check(rc == CGT_AMD_OK, "LayerNorm: %s", cgt_amd_last_error());
            }"""
        return core.NativeCompileInfo(code, includes=["cgt_amd.h"], closure_triples=[("eps", ctypes.c_double, self.eps)],
                                      gpu_deref_mask=(True, True, True))


class LayerNormBackward(core.Op):
    """inputs [x, gamma, mean, rstd, gy] -> (gx, ggamma, gbeta)."""
    available_impls = ("native_gpu",)

    def typ_apply(self, input_types):
        _check_operands("LayerNormBackward", input_types, [1], [4])
        return core.TupleType(input_types[0], input_types[1], input_types[1])

    def shp_apply(self, inputs):
        _check_shapes("LayerNormBackward", inputs[0], inputs[1:2], inputs[4:5])
        return tuple(core.shape(inputs[i]) for i in (0, 1, 1))

    def get_native_compile_info(self, input_types, devtype):
        assert devtype == "gpu"
        code = r"""
            CGT_EXPORT_C void $function(void* cl, cgtArray** reads, cgtTuple* write) {
                cgtArray *X = reads[0], *gamma = reads[1], *mean = reads[2], *rstd = reads[3], *gy = reads[4];
                cgtArray *gx = (cgtArray*)write->getitem(0), *ggamma = (cgtArray*)write->getitem(1), *gbeta = (cgtArray*)write->getitem(2);
""" + _ROWS + r"""
                cgt_check(gamma->size() == cols && mean->size() == rows && rstd->size() == rows && gy->size() == X->size() &&
                          gx->size() == X->size() && ggamma->size() == cols && gbeta->size() == cols,
                          "LayerNormBackward: operands do not fit the input");
                if (cgtGlobalStatus != cgtStatusOK) return;
                int rc = cgt_amd_layer_norm_bwd_f32((const float*)X->data(), (const float*)gamma->data(), (const float*)mean->data(),
                    (const float*)rstd->data(), (const float*)gy->data(), rows, cols, (float*)gx->data(), (float*)ggamma->data(),
                    (float*)gbeta->data(), cgt_get_stream());
                cgt_check(rc == CGT_AMD_OK, "LayerNormBackward: %s", cgt_amd_last_error());
            }"""
        return core.NativeCompileInfo(code, includes=["cgt_amd.h"], gpu_deref_mask=(True,) * 5)


class DropoutAddLayerNorm(core.Op):
    """inputs [x, residual, gamma, beta] (+ [rng] when p > 0) -> (y, h, mean, rstd): h = residual + dropout(x),
    y = layer norm of h."""
    available_impls = ("native_gpu",)

    def __init__(self, p, eps, channel):
        self.p, self.eps, self.channel = float(p), float(eps), int(channel)
        if not 0 <= self.channel < 1 << 32:
            raise ValueError("channel must be a whole number of 32 bits (got %s)" % (channel,))

    def get_diff(self, num_inputs):
        return [True] * 4 + [False] * (num_inputs - 4)

    def typ_apply(self, input_types):
        _check_operands("DropoutAddLayerNorm", input_types, [2, 3], [1])
        from .dropout import check_rng
        if self.p:
            check_rng(input_types[4])
        x = input_types[0]
        stat = core.TensorType("f4", x.ndim - 1)
        return core.TupleType(x, x, stat, stat)

    def shp_apply(self, inputs):
        _check_shapes("DropoutAddLayerNorm", inputs[0], inputs[2:4], inputs[1:2])
        s = core.shape(inputs[0])
        return (s, s, s[:-1], s[:-1])

    def pullback(self, inputs, output, gout):
        from .dropout import Dropout
        _y, h, mean, rstd = core.unpack(output)
        if any(g is not None for g in gout[2:]):
            raise core.MethodNotDefined("DropoutAddLayerNorm: gradients go through y and h, not through the statistics")
        gy, gh = gout[:2]
        rng = list(inputs[4:])
        if gy is None:          # only h was used: the residual add and the dropout alone
            return [core.Result(Dropout(self.p, self.channel), [gh] + rng) if self.p else gh, gh, None, None] + [None] * len(rng)
        g = core.unpack(core.Result(DropoutAddLayerNormBackward(self.p, self.channel, gh is not None),
                                    [h, inputs[2], mean, rstd, gy] + ([gh] if gh is not None else []) + rng))
        if not self.p:
            g = [g[0]] + g
        return g + [None] * len(rng)

    def get_native_compile_info(self, input_types, devtype):
        assert devtype == "gpu"
        code = r"""
            CGT_EXPORT_C void $function($closure* cl, cgtArray** reads, cgtTuple* write) {
                cgtArray *X = reads[0], *res = reads[1], *gamma = reads[2], *beta = reads[3], *rng = cl->p > 0 ? reads[4] : NULL;
                cgtArray *y = (cgtArray*)write->getitem(0), *h = (cgtArray*)write->getitem(1);
                cgtArray *mean = (cgtArray*)write->getitem(2), *rstd = (cgtArray*)write->getitem(3);
""" + _ROWS + r"""
                cgt_check(res->size() == X->size() && gamma->size() == cols && beta->size() == cols && (!rng || rng->size() == 2) &&
                          y->size() == X->size() && h->size() == X->size() && mean->size() == rows && rstd->size() == rows,
                          "DropoutAddLayerNorm: residual, weights, generator state or outputs do not fit the input");
                if (cgtGlobalStatus != cgtStatusOK) return;
                int rc = cgt_amd_dropout_add_layer_norm_fwd_f32((const float*)X->data(), (const float*)res->data(), rows, cols, cl->p,
                    rng ? (const long long*)rng->data() : NULL, (unsigned)cl->channel, (const float*)gamma->data(), (const float*)beta->data(),
                    cl->eps, (float*)y->data(), (float*)h->data(), (float*)mean->data(), (float*)rstd->data(), cgt_get_stream());
                cgt_check(rc == CGT_AMD_OK, "DropoutAddLayerNorm: %s", cgt_amd_last_error());
            }"""
        triples = [("p", ctypes.c_double, self.p), ("eps", ctypes.c_double, self.eps), ("channel", ctypes.c_long, self.channel)]
        return core.NativeCompileInfo(code, includes=["cgt_amd.h"], closure_triples=triples, gpu_deref_mask=(True,) * len(input_types))


class DropoutAddLayerNormBackward(core.Op):
    """inputs [h, gamma, mean, rstd, gy] (+ [gh] when has_gh) (+ [rng] when p > 0) -> (gx, gresidual, ggamma, gbeta);
    without gx when p is 0, where it equals gresidual."""
    available_impls = ("native_gpu",)

    def __init__(self, p, channel, has_gh):
        self.p, self.channel, self.has_gh = float(p), int(channel), bool(has_gh)

    def typ_apply(self, input_types):
        _check_operands("DropoutAddLayerNormBackward", input_types, [1], [4] + ([5] if self.has_gh else []))
        h, gamma = input_types[:2]
        return core.TupleType(*([h] if self.p else []), h, gamma, gamma)

    def shp_apply(self, inputs):
        _check_shapes("DropoutAddLayerNormBackward", inputs[0], inputs[1:2], inputs[4:6] if self.has_gh else inputs[4:5])
        h, gamma = core.shape(inputs[0]), core.shape(inputs[1])
        return tuple(([h] if self.p else []) + [h, gamma, gamma])

    def get_native_compile_info(self, input_types, devtype):
        assert devtype == "gpu"
        code = r"""
            CGT_EXPORT_C void $function($closure* cl, cgtArray** reads, cgtTuple* write) {
                cgtArray *X = reads[0], *gamma = reads[1], *mean = reads[2], *rstd = reads[3], *gy = reads[4];
                cgtArray *gh = cl->has_gh ? reads[5] : NULL, *rng = cl->p > 0 ? reads[5 + cl->has_gh] : NULL;
                int at = 0;
                cgtArray *gx = cl->p > 0 ? (cgtArray*)write->getitem(at++) : NULL;
                cgtArray *gres = (cgtArray*)write->getitem(at++), *ggamma = (cgtArray*)write->getitem(at++), *gbeta = (cgtArray*)write->getitem(at);
""" + _ROWS + r"""
                cgt_check(gamma->size() == cols && mean->size() == rows && rstd->size() == rows && gy->size() == X->size() &&
                          (!gh || gh->size() == X->size()) && (!rng || rng->size() == 2) && (!gx || gx->size() == X->size()) &&
                          gres->size() == X->size() && ggamma->size() == cols && gbeta->size() == cols,
                          "DropoutAddLayerNormBackward: operands do not fit the input");
                if (cgtGlobalStatus != cgtStatusOK) return;
                int rc = cgt_amd_dropout_add_layer_norm_bwd_f32((const float*)X->data(), (const float*)gamma->data(), (const float*)mean->data(),
                    (const float*)rstd->data(), (const float*)gy->data(), gh ? (const float*)gh->data() : NULL, rows, cols, cl->p,
                    rng ? (const long long*)rng->data() : NULL, (unsigned)cl->channel, gx ? (float*)gx->data() : NULL,
                    (float*)gres->data(), (float*)ggamma->data(), (float*)gbeta->data(), cgt_get_stream());
                cgt_check(rc == CGT_AMD_OK, "DropoutAddLayerNormBackward: %s", cgt_amd_last_error());
            }"""
        triples = [("p", ctypes.c_double, self.p), ("channel", ctypes.c_long, self.channel), ("has_gh", ctypes.c_int, int(self.has_gh))]
        return core.NativeCompileInfo(code, includes=["cgt_amd.h"], closure_triples=triples, gpu_deref_mask=(True,) * len(input_types))


def layer_norm(x, gamma, beta, eps=1e-5):
    """gamma * (x - mean) / sqrt(var + eps) + beta over the last axis of x."""
    return core.Result(LayerNorm(eps), [x, gamma, beta])[0]


def dropout_add_layer_norm(x, residual, gamma, beta, p=0.0, rng=None, channel=0, eps=1e-5):
    """(y, h): h = residual + dropout(x), y = layer_norm(h), in one pass each way."""
    from .dropout import rng_node, resolved
    p = resolved(p)
    out = core.Result(DropoutAddLayerNorm(p, eps, channel), [x, residual, gamma, beta] + ([rng_node(rng)] if p else []))
    y, h = core.unpack(out)[:2]
    return y, h
