"""Attention with a learned relative position bias, as tuple-valued ops over the fused kernels.

The reference has no counterpart; the composition these replace is BatchedMul22 -> bias add -> softmax ->
BatchedMul22 over an array of scores that these never store.
"""
import ctypes
from collections import namedtuple

import numpy as np

from .. import core
from .dropout import check_rng, resolved, rng_node

AttentionInfo = namedtuple("AttentionInfo", ["scale", "causal", "bidirectional", "max_distance", "q_offset", "p", "channel", "layout",
                                             "has_table", "has_q_lengths", "has_k_lengths", "has_q_offsets",
                                             "scale_by_width"])
AttentionInfo.__new__.__defaults__ = (0, 0)


def make_closure(info):
    return [
        ("scale", ctypes.c_double, info.scale),
        ("p", ctypes.c_double, info.p),
        ("max_distance", ctypes.c_long, info.max_distance),
        ("q_offset", ctypes.c_long, info.q_offset),
        ("channel", ctypes.c_long, info.channel),
        ("causal", ctypes.c_int, info.causal),
        ("bidirectional", ctypes.c_int, info.bidirectional),
        ("layout", ctypes.c_int, info.layout),
        ("has_table", ctypes.c_int, info.has_table),
        ("has_q_lengths", ctypes.c_int, info.has_q_lengths),
        ("has_k_lengths", ctypes.c_int, info.has_k_lengths),
        ("has_q_offsets", ctypes.c_int, info.has_q_offsets),
        ("scale_by_width", ctypes.c_int, info.scale_by_width),
    ]


# the operands both directions start with: q, k, v, then those of table, q_lengths, k_lengths, q_offsets, rng that exist
_OPERANDS = r"""
                cgtArray *q = reads[0], *k = reads[1], *v = reads[2];
                int at = 3;
                cgtArray *table = cl->has_table ? reads[at++] : NULL, *qn = cl->has_q_lengths ? reads[at++] : NULL;
                cgtArray *kn = cl->has_k_lengths ? reads[at++] : NULL, *qo = cl->has_q_offsets ? reads[at++] : NULL;
                cgtArray *rng = cl->p > 0 ? reads[at++] : NULL;
                const int t = cl->layout ? 1 : 2;
                // D^-1/2 of the arrays at hand: a compiled function serves any head width
                const double scale = cl->scale_by_width && q->shape()[3] ? 1.0 / sqrt((double)q->shape()[3]) : cl->scale;
                const long B = q->shape()[0], H = q->shape()[3 - t], Tq = q->shape()[t], D = q->shape()[3], Tk = k->shape()[t];
                cgt_check(k->size() == B * H * Tk * D && k->shape()[3 - t] == H && k->shape()[3] == D && v->size() == k->size() &&
                          (!table || (table->ndim() == 2 && table->shape()[1] == H)) && (!qn || (qn->size() == B && qn->dtype() == cgt_i4)) &&
                          (!kn || (kn->size() == B && kn->dtype() == cgt_i4)) && (!qo || (qo->size() == B && qo->dtype() == cgt_i4)) &&
                          (!rng || rng->size() == 2),
                          "RelativeAttention: operands do not fit each other");
"""

def _call(name, before, after):
    """The call of one of the two forms of an entry point: one position for all sequences, or an array of them."""
    both = []
    for form, position in (("_at", "(const int*)qo->data()"), ("", "cl->q_offset")):
        both.append("cgt_amd_rel_attention" + form + "_" + name + "_f32(" + before + r""", B, H, Tq, Tk, D, cl->layout, table ? table->shape()[0] : 0,
                    cl->bidirectional, cl->max_distance, scale, cl->causal, """ + position + r""", qn ? (const int*)qn->data() : NULL,
                    kn ? (const int*)kn->data() : NULL, cl->p, rng ? (const long long*)rng->data() : NULL, (unsigned)cl->channel,
                    """ + after + ", cgt_get_stream())")
    return "qo ? " + both[0] + "\n                  : " + both[1]


def _check_types(info, types):
    assert all(t == core.TensorType("f4", 4) for t in types[:3]), "RelativeAttention takes q, k and v of four axes, float32"
    rest = list(types[3:])
    if info.has_table:
        assert rest.pop(0) == core.TensorType("f4", 2), "RelativeAttention: the bias table is a float32 matrix [buckets, heads]"
    for has in (info.has_q_lengths, info.has_k_lengths, info.has_q_offsets):
        if has:
            assert rest.pop(0) == core.TensorType("i4", 1), "RelativeAttention: lengths and offsets are int32 arrays of one axis"
    if info.p:
        check_rng(rest.pop(0))


def _check_shapes(info, inputs):
    q, k, v = (core.shape(i) for i in inputs[:3])
    t = 1 if info.layout else 2
    if v != k or (k[0], k[3 - t], k[3]) != (q[0], q[3 - t], q[3]):
        raise ValueError("RelativeAttention: q %s, k %s and v %s do not fit each other" % (q, k, v))
    rest = list(inputs[3:])
    if info.has_table and core.shape(rest.pop(0))[1] != q[3 - t]:
        raise ValueError("RelativeAttention: the bias table must have a column for each of the %d heads" % q[3 - t])
    for has in (info.has_q_lengths, info.has_k_lengths, info.has_q_offsets):
        if has and core.shape(rest.pop(0)) != q[:1]:
            raise ValueError("RelativeAttention: one length or offset for each of the %d sequences" % q[0])


class RelativeAttention(core.Op):
    """inputs [q, k, v] (+ [table]) (+ [q_lengths]) (+ [k_lengths]) (+ [q_offsets]) (+ [rng] when p > 0) -> (o, lse)."""
    available_impls = ("native_gpu",)

    def __init__(self, info):
        assert isinstance(info, AttentionInfo)
        self.info = info

    def get_diff(self, num_inputs):
        n = 3 + self.info.has_table
        return [True] * n + [False] * (num_inputs - n)

    def typ_apply(self, input_types):
        _check_types(self.info, input_types)
        return core.TupleType(input_types[0], core.TensorType("f4", 3))

    def shp_apply(self, inputs):
        _check_shapes(self.info, inputs)
        s = core.shape(inputs[0])
        t = 1 if self.info.layout else 2
        return (s, [s[0], s[3 - t], s[t]])

    def pullback(self, inputs, output, gout):
        if gout[1] is not None or gout[0] is None:
            raise core.MethodNotDefined("RelativeAttention: gradients go through o only, not through lse")
        o, lse = core.unpack(output)
        g = core.unpack(core.Result(RelativeAttentionBackward(self.info), list(inputs) + [o, lse, gout[0]]))
        return g + [None] * (len(inputs) - len(g))

    def get_native_compile_info(self, input_types, devtype):
        assert devtype == "gpu"
        code = r"""
            CGT_EXPORT_C void $function($closure* cl, cgtArray** reads, cgtTuple* write) {
""" + _OPERANDS + r"""
                cgtArray *o = (cgtArray*)write->getitem(0), *lse = (cgtArray*)write->getitem(1);
                cgt_check(o->size() == q->size() && lse->size() == B * H * Tq, "RelativeAttention: outputs do not fit the input");
                if (cgtGlobalStatus != cgtStatusOK) return;
                int rc = """ + _call("fwd", "(const float*)q->data(), (const float*)k->data(), (const float*)v->data(), "
                                     "table ? (const float*)table->data() : NULL", "(float*)o->data(), (float*)lse->data()") + r""";
                cgt_check(rc == CGT_AMD_OK, "RelativeAttention: %s", cgt_amd_last_error());
            }"""
        return core.NativeCompileInfo(code, includes=["math.h", "cgt_amd.h"], closure_triples=make_closure(self.info),
                                      gpu_deref_mask=(True,) * len(input_types))


class RelativeAttentionBackward(core.Op):
    """The inputs of RelativeAttention, its results and the cotangent of o -> (gq, gk, gv) (+ (gtable,))."""
    available_impls = ("native_gpu",)

    def __init__(self, info):
        self.info = info

    def typ_apply(self, input_types):
        _check_types(self.info, input_types)
        return core.TupleType(*input_types[:3 + self.info.has_table])

    def shp_apply(self, inputs):
        _check_shapes(self.info, inputs)
        if core.shape(inputs[-1]) != core.shape(inputs[0]):
            raise ValueError("RelativeAttentionBackward: the cotangent %s must have q's shape %s" % (core.shape(inputs[-1]), core.shape(inputs[0])))
        return tuple(core.shape(i) for i in inputs[:3 + self.info.has_table])

    def get_native_compile_info(self, input_types, devtype):
        assert devtype == "gpu"
        code = r"""
            CGT_EXPORT_C void $function($closure* cl, cgtArray** reads, cgtTuple* write) {
""" + _OPERANDS + r"""
                cgtArray *o = reads[at], *lse = reads[at + 1], *go = reads[at + 2];
                cgtArray *gq = (cgtArray*)write->getitem(0), *gk = (cgtArray*)write->getitem(1), *gv = (cgtArray*)write->getitem(2);
                cgtArray *gtable = table ? (cgtArray*)write->getitem(3) : NULL;
                cgt_check(o->size() == q->size() && go->size() == q->size() && lse->size() == B * H * Tq && gq->size() == q->size() &&
                          gk->size() == k->size() && gv->size() == k->size() && (!gtable || gtable->size() == table->size()),
                          "RelativeAttentionBackward: operands do not fit the input");
                if (cgtGlobalStatus != cgtStatusOK) return;
                int rc = """ + _call("bwd", "(const float*)q->data(), (const float*)k->data(), (const float*)v->data(), "
                                     "table ? (const float*)table->data() : NULL, (const float*)o->data(), (const float*)lse->data(), (const float*)go->data()",
                                     "(float*)gq->data(), (float*)gk->data(), (float*)gv->data(), gtable ? (float*)gtable->data() : NULL") + r""";
                cgt_check(rc == CGT_AMD_OK, "RelativeAttentionBackward: %s", cgt_amd_last_error());
            }"""
        return core.NativeCompileInfo(code, includes=["math.h", "cgt_amd.h"], closure_triples=make_closure(self.info),
                                      gpu_deref_mask=(True,) * len(input_types))


def _lengths_node(lengths):
    """int32 [B] on the device: the sequences' lengths or offsets."""
    if isinstance(lengths, core.Node) or isinstance(lengths, core.GpuArray):
        return core.as_node(lengths)
    lengths = np.asarray(lengths)
    if lengths.dtype.kind not in "iu":
        raise TypeError("lengths and offsets are whole numbers, got %s" % lengths.dtype)
    return core.as_node(core.to_gpu(lengths.astype(np.int32)))


def relative_attention(q, k, v, table=None, scale=None, causal=False, bidirectional=None, max_distance=128, q_offset=0,
                       q_lengths=None, k_lengths=None, p=0.0, rng=None, channel=0, layout="bhtd"):
    """softmax(scale * q k^T + table[bucket(key - query position)]) v per sequence and head.

    q [B,H,Tq,D], k and v [B,H,Tk,D] (layout "bthd": [B,T,H,D], as a projection leaves them), table [buckets, H].
    scale is D^-1/2 and bidirectional `not causal` unless given.  Lengths (int32 [B]) describe a padded batch.
    q_offset is the position of the first query among the keys: a number, or int32 [B] with one for each sequence
    (q_offset = k_lengths - Tq for new tokens at the ends of sequences of different lengths).  Lengths and such offsets are inputs of the op:
    a compiled function that takes them as arguments steps through a cache of fixed size.
    p, rng and channel drop values of the softmax as nn.dropout would."""
    q, k, v = (core.as_node(x) for x in (q, k, v))
    if layout not in ("bhtd", "bthd"):
        raise ValueError("layout is 'bhtd' or 'bthd' (got %r)" % (layout,))
    if q.ndim != 4:
        raise ValueError("attention takes q, k and v of four axes (got %d)" % q.ndim)
    p = resolved(p)
    if not 0 <= int(channel) < 1 << 32:
        raise ValueError("channel must be a whole number of 32 bits (got %s)" % (channel,))
    each = isinstance(q_offset, (core.Node, core.GpuArray)) or np.ndim(q_offset) > 0
    info = AttentionInfo(float(0.0 if scale is None else scale), int(bool(causal)),
                         int(bool(not causal if bidirectional is None else bidirectional)), int(max_distance), 0 if each else int(q_offset), p, int(channel),
                         int(layout == "bthd"), int(table is not None), int(q_lengths is not None), int(k_lengths is not None), int(each),
                         int(scale is None))
    inputs = [q, k, v] + ([core.as_node(table)] if table is not None else [])
    inputs += [_lengths_node(n) for n in (q_lengths, k_lengths, q_offset if each else None) if n is not None] + ([rng_node(rng)] if p else [])
    result = core.Result(RelativeAttention(info), inputs)
    # numbers that were computed from extents (q_offset = Tk - Tq) tie a compiled function to the shapes it was traced with
    for n in (max_distance,) if each else (q_offset, max_distance):
        if isinstance(n, core.ShapeInt) and not n.is_constant():
            result.baked_expr = ("+", result.baked_expr, n.expr) if result.shape_baked else n.expr
            result.shape_baked = True
    return result[0]
