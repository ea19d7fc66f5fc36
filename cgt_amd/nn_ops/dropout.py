"""Dropout from a counter-based generator.

The mask is a function of (seed, step, channel, element), formed again in the gradient and never stored.  `rng` is
an int64 array (seed, step); it is an input of the op, not part of its closure, so a compiled function that takes
it as an argument, or a captured graph whose copy of it is rewritten, draws new masks at every step.
"""
import ctypes

import numpy as np

from .. import core
from ..gpuarray import GpuArray, to_gpu


def resolved(p):
    """The probability if the generator's 16-bit numbers resolve it, 0.0 if it rounds to nothing."""
    p = float(p)
    if not 0.0 <= p < 1.0 - 2.0 ** -17:
        raise ValueError("the dropout probability must be at least 0 and below 1 by 2^-16 or more (got %g)" % p)
    return p if p * 65536.0 + 0.5 >= 1.0 else 0.0


def rng_node(rng):
    """The generator's state as a node: int64 [seed, step]."""
    if rng is None:
        raise ValueError("dropout needs the generator's state: an int64 array (seed, step)")
    if not isinstance(rng, core.Node):
        if not isinstance(rng, GpuArray):
            rng = np.asarray(rng)
            if rng.dtype.kind not in "iu":
                raise TypeError("the generator's state is an int64 array (seed, step), got %s" % rng.dtype)
            rng = to_gpu(rng.astype(np.int64))
        rng = core.constant(rng)
    check_rng(rng.typ)
    if tuple(rng.shape) != (2,):
        raise ValueError("the generator's state has two elements, seed and step (got shape %s)" % (tuple(rng.shape),))
    return rng


def check_rng(typ):
    if typ != core.TensorType("i8", 1):
        raise TypeError("the generator's state is an int64 array (seed, step), got %s" % typ)


class Dropout(core.Op):
    """inputs [x, rng] (+ [residual]) -> x * keep / share kept (+ residual)."""
    available_impls = ("native_gpu",)

    def __init__(self, p, channel):
        self.p, self.channel = float(p), int(channel)
        if not 0 <= self.channel < 1 << 32:
            raise ValueError("channel must be a whole number of 32 bits (got %s)" % (channel,))

    def get_diff(self, num_inputs):
        return [True, False, True][:num_inputs]

    def typ_apply(self, input_types):
        assert input_types[0].dtype == "f4", "Dropout takes a float32 array"
        check_rng(input_types[1])
        assert len(input_types) == 2 or input_types[2] == input_types[0], "Dropout: the residual must be an array like x"
        return input_types[0]

    def shp_apply(self, inputs):
        s = core.shape(inputs[0])
        if len(inputs) > 2 and core.shape(inputs[2]) != s:
            raise ValueError("Dropout: mismatched shapes %s %s" % (s, core.shape(inputs[2])))
        return s

    def pullback(self, inputs, output, gout):
        return self.pullback_wanted(inputs, output, gout, self.get_diff(len(inputs)))

    def pullback_wanted(self, inputs, output, gout, wanted):
        gx = core.Result(Dropout(self.p, self.channel), [gout, inputs[1]]) if wanted[0] else None
        return [gx, None] + ([gout] if len(inputs) > 2 else [])

    def get_native_compile_info(self, input_types, devtype):
        assert devtype == "gpu"
        code = r"""
            CGT_EXPORT_C void $function($closure* cl, cgtArray** reads, cgtArray* write) {
                cgtArray *X = reads[0], *rng = reads[1], *res = cl->has_residual ? reads[2] : NULL;
                cgt_check(rng->size() == 2 && write->size() == X->size() && (!res || res->size() == X->size()),
                          "Dropout: generator state, residual or output do not fit the input");
                if (cgtGlobalStatus != cgtStatusOK) return;
                int rc = cgt_amd_dropout_f32((const float*)X->data(), res ? (const float*)res->data() : NULL, X->size(), cl->p,
                    (const long long*)rng->data(), (unsigned)cl->channel, (float*)write->data(), cgt_get_stream());
                cgt_check(rc == CGT_AMD_OK, "Dropout: %s", cgt_amd_last_error());
            }"""
        triples = [("p", ctypes.c_double, self.p), ("channel", ctypes.c_long, self.channel),
                   ("has_residual", ctypes.c_int, int(len(input_types) > 2))]
        return core.NativeCompileInfo(code, includes=["cgt_amd.h"], closure_triples=triples, gpu_deref_mask=(True,) * len(input_types))


def dropout(x, p, rng, channel=0, residual=None):
    """x with each element dropped with probability p and the kept ones divided by the share kept, plus `residual`
    if given.  Different layers take different `channel`s; different steps, different rng = (seed, step)."""
    x = core.as_node(x)
    p = resolved(p)
    if p == 0.0:
        return x if residual is None else x + core.as_node(residual)
    return core.Result(Dropout(p, channel), [x, rng_node(rng)] + ([] if residual is None else [residual]))


def rng_state(seed, step=0):
    """The generator's state as a device array: int64 [seed, step]."""
    return to_gpu(np.array([seed, step], np.int64))
