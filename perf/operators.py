"""Operators for training and serving nets with language-model heads, as measurable cases.

Three operators that meet in one training step, called through the public binding (``eddl_b200.capi``, the C ABI of
``include/eddl_b200.h``):

``fp8``      dense products in 8-bit floating point with an fp32 scale for each block of 128 values along the reduction: the
             quantisation (``fp8_quantize``), the product (``fp8_mult2d``), and the three products of a training step.
``norm``     what stands between two blocks of a residual net: normalise the block's output, scale it by a gate, add it to the scaled
             residual stream and normalise the sum for the next block (``norm_residual_fwd`` / ``norm_residual_bwd``).
``distill``  the loss of a student against a teacher's top logits, mixed with the cross-entropy of hard labels, and its gradient
             with respect to the student's logits (``distill``).

Matrices in 8 bits have rows of a pitch that is a multiple of 16 bytes; scale [b][r] belongs to columns 128 b .. 128 b + 127 of
row r, or of the rows 128 r .. 128 r + 127 where a block has 128 rows.  A scale is the block's largest magnitude over the largest
number of the format, or the next power of two from there on: then nothing but the 8 bits themselves is rounded.
"""
import math

import torch

own = False
DEV = 0
DEVICE = "cuda:%d" % DEV
BLOCK = 128
FORMATS = {"e4m3": (0, torch.float8_e4m3fn, 448.0, 3, -6), "e5m2": (1, torch.float8_e5m2, 57344.0, 2, -14)}      # code, type, largest, mantissa bits, least exponent
SMALLEST = 2.0 ** -100          # a block whose largest magnitude is below this is scaled as if it were this


# ---- the cases -------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token through a dense layer whose weights were quantised once: the weights' bytes and latency are all there is
        _product(1, 4096, 4096, 128, name="fp8_product_one_token"),
        # a handful of sequences that answer together, rows and columns that end inside a block
        _product(24, 5000, 2056, 128, name="fp8_product_24_tokens"),
        # a large batch of activations against the weights: the arithmetic decides
        _product(8192, 8192, 8192, 128, name="fp8_product_8192"),
        # activations on their way into a product: both directions in one pass, for the forward pass and the weights' gradient
        _quantize(8192, 4096, 1, "e4m3", False, name="fp8_quantize_8192x4096"),
        # a training step of the classifier head of ResNet-50 at the headline batch: small products, so launches decide
        _dense(64, 1000, 2048, "e4m3", name="fp8_dense_head_64x1000"),
        # a training step of a square dense layer over a few thousand tokens, output gradients in the format with more range
        _dense(4096, 4096, 4096, "e5m2", name="fp8_dense_4096"),
        # one image's worth of tokens between two blocks, answering
        _norm(1, 49, 768, "rms", "group", 1, False, name="norm_answer_49x768"),
        # a batch of images as 196 tokens each, a gate of its own for each image, training
        _norm(64, 196, 768, "layer", "group", 1, True, name="norm_images_64x196x768"),
        # a wide net's tokens, one gate for each channel, training
        _norm(1, 12288, 4096, "rms", "group", 1, True, name="norm_tokens_12288x4096"),
        # an image classifier's student: a thousand classes, the teacher's ten best
        _distill(64, 1000, 0, 10, 4.0, 0.5, False, name="distill_64x1000_top10"),
        # a language model's student: an ordinary vocabulary
        _distill(4096, 32000, 0, 64, 2.0, 0.3, False, name="distill_4096x32000_top64"),
        # a large odd vocabulary in padded rows, the rest of the teacher's mass as a class of its own, some rows masked out
        _distill(1023, 131071, 1, 128, 1.0, 0.0, True, name="distill_1023x131071_top128"),
    ]


def _product(m, n, k, block_b, format_a="e4m3", **more):
    return dict(more, op="fp8_product", m=m, n=n, k=k, block_b=block_b, format_a=format_a)


def _quantize(rows, cols, block_rows, form, pow2, **more):
    return dict(more, op="fp8_quantize", rows=rows, cols=cols, block_rows=block_rows, format=form, pow2=pow2)


def _dense(m, n, k, form, **more):
    return dict(more, op="fp8_dense", m=m, n=n, k=k, format=form)


def _norm(groups, rows, cols, kind, gate, post, train, **more):
    return dict(more, op="norm", groups=groups, rows=rows, cols=cols, kind=kind, gate=gate, post=post, train=train)


def _distill(rows, cols, pad, k, temperature, alpha, tail, **more):
    return dict(more, op="distill", rows=rows, cols=cols, pad=pad, k=k, temperature=temperature, alpha=alpha, tail=tail)


def _log_int(rng, lo, hi):
    """A whole number whose logarithm is uniform over [lo, hi]: odd ones come as often as even ones."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges."""
    what = rng.choice(["fp8_product", "fp8_product", "fp8_quantize", "fp8_dense", "norm", "norm", "distill", "distill"])
    if what == "fp8_product":
        while True:
            m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 64, 8192), _log_int(rng, 64, 8192)
            if m * n * k <= 2 ** 39:
                return _product(m, n, k, rng.choice([128, 128, 1]), rng.choice(["e4m3", "e4m3", "e5m2"]))
    if what == "fp8_quantize":
        while True:
            rows, cols = _log_int(rng, 1, 16384), _log_int(rng, 64, 16384)
            if rows * cols <= 2 ** 25:
                return _quantize(rows, cols, rng.choice([1, 1, 128]), rng.choice(["e4m3", "e5m2"]), rng.random() < 0.5)
    if what == "fp8_dense":
        while True:
            m, n, k = _log_int(rng, 16, 8192), _log_int(rng, 10, 8192), _log_int(rng, 64, 8192)
            if m * n * k <= 2 ** 36:
                return _dense(m, n, k, rng.choice(["e4m3", "e5m2"]))
    if what == "norm":
        while True:
            groups, rows, cols = _log_int(rng, 1, 256), _log_int(rng, 1, 4096), _log_int(rng, 64, 16384)
            if groups * rows * cols <= 2 ** 25:
                return _norm(groups, rows, cols, rng.choice(["rms", "layer"]), rng.choice(["group", "group", "none"]), rng.choice([1, 1, 0]), rng.random() < 0.7)
    while True:
        rows, cols = _log_int(rng, 1, 8192), _log_int(rng, 10, 131072)
        if rows * cols <= 2 ** 27:
            tail = rng.random() < 0.4
            return _distill(rows, cols, rng.choice([0, 0, 1, 5, 64]), min(_log_int(rng, 1, 256), cols // 2), rng.choice([0.7, 1.0, 2.0, 4.0]), rng.choice([0.0, 0.3, 0.5]), tail)


# ---- inputs ------------------------------------------------------------------------------------------------------------------
class _Random:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEVICE)
        self.g.manual_seed(int(seed))

    def normal(self, *shape, scale=1.0, shift=0.0):
        return torch.empty(shape, device=DEVICE).normal_(shift, scale, generator=self.g)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.empty(shape, device=DEVICE).uniform_(lo, hi, generator=self.g)

    def matrix(self, rows, cols, scale):
        """Values as a layer's input has them: most rows alike, a few channels several times as large."""
        return self.normal(rows, cols, scale=scale) * torch.exp(self.normal(1, cols, scale=0.5))

    def whole(self, hi, *shape):
        return torch.randint(0, hi, shape, generator=self.g, device=DEVICE)


def _pitch(cols):
    return (cols + 15) // 16 * 16


def _blocks(n, size=BLOCK):
    return (n + size - 1) // size


class _Eight:
    """Room for a matrix in 8 bits with its scales."""

    def __init__(self, rows, cols, form, block_rows):
        self.rows, self.cols, self.form, self.block_rows = rows, cols, form, block_rows
        self.store = torch.zeros((rows, _pitch(cols)), device=DEVICE, dtype=torch.uint8).view(FORMATS[form][1])
        self.scale = torch.zeros((_blocks(cols), _blocks(rows, block_rows)), device=DEVICE)

    @property
    def q(self):
        return self.store[:, :self.cols]

    def fill(self, a):
        q, scale = _plain_quantize(a, self.form, self.block_rows, False)
        self.store.view(torch.uint8)[:, :self.cols] = q.view(torch.uint8)
        self.scale.copy_(scale)
        return self

    def args(self):
        return self.store.data_ptr(), self.store.shape[1], self.scale.data_ptr(), FORMATS[self.form][0], self.block_rows


def _ids(rand, logits, k):
    best = torch.topk(logits, k, dim=1)
    return best.indices.to(torch.int32).contiguous(), best.values.contiguous()


def prepare(case, seed):
    rand, op, s = _Random(seed), case["op"], {"case": case}
    if op == "fp8_product":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"] = _Eight(m, k, case["format_a"], 1).fill(rand.matrix(m, k, 1.0))
        s["b"] = _Eight(n, k, "e4m3", case["block_b"]).fill(rand.matrix(n, k, 0.05))
        s["c"] = torch.zeros((m, n), device=DEVICE)
    elif op == "fp8_quantize":
        rows, cols = case["rows"], case["cols"]
        s["a"] = rand.matrix(rows, cols, 1.0)
        s["q"], s["qt"] = _Eight(rows, cols, case["format"], case["block_rows"]), _Eight(cols, rows, case["format"], case["block_rows"])
    elif op == "fp8_dense":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"], s["w"], s["dy"] = rand.matrix(m, k, 1.0), rand.matrix(n, k, 0.05), rand.matrix(m, n, 1e-3)
        s["xq"], s["xt"] = _Eight(m, k, "e4m3", 1), _Eight(k, m, "e4m3", 1)
        s["wq"], s["wt"] = _Eight(n, k, "e4m3", 128), _Eight(k, n, "e4m3", 128)
        s["dq"], s["dt"] = _Eight(m, n, case["format"], 1), _Eight(n, m, case["format"], 1)
        s["y"], s["dx"], s["dw"] = (torch.zeros(shape, device=DEVICE) for shape in ((m, n), (m, k), (n, k)))
    elif op == "norm":
        groups, rows, cols = case["groups"], case["rows"], case["cols"]
        total, layer, train = groups * rows, case["kind"] == "layer", case["train"]
        s["f"], s["r"] = rand.normal(total, cols, scale=0.7, shift=0.1), rand.normal(total, cols, scale=1.5)
        s["gate"] = rand.normal(groups, cols, scale=0.3, shift=0.5) if case["gate"] == "group" else None
        s["g1"] = rand.normal(cols, scale=0.1, shift=1.0) if case["post"] else None
        s["b1"] = rand.normal(cols, scale=0.1) if case["post"] and layer else None
        s["g2"], s["b2"] = rand.normal(cols, scale=0.1, shift=1.0), rand.normal(cols, scale=0.1) if layer else None
        s["res_scale"], s["eps"] = 0.9, 1e-5
        names = ["r_out", "h"]
        if train:
            s["dh"], s["dr_out"] = rand.normal(total, cols, scale=1e-2), rand.normal(total, cols, scale=1e-2)
            names += ["df", "dr"]
        for name in names:
            s[name] = torch.zeros((total, cols), device=DEVICE)
        s["stats"] = torch.zeros((total, 4), device=DEVICE) if train else None
        for name, of in (("dgate", "gate"), ("dg1", "g1"), ("db1", "b1"), ("dg2", "g2"), ("db2", "b2")):
            s[name] = torch.zeros_like(s[of]) if train and s[of] is not None else None
    else:
        rows, cols, k, temperature = case["rows"], case["cols"], case["k"], case["temperature"]
        ld = cols + case["pad"]
        s["logits"] = rand.normal(rows, ld, scale=2.0)
        teacher = s["logits"][:, :cols] * 0.7 + rand.normal(rows, cols, scale=2.0)
        s["ids"], s["teacher"] = _ids(rand, teacher, k)
        s["teacher_lse"] = torch.logsumexp(teacher.double() / temperature, 1).float() if case["tail"] else None
        s["labels"] = s["ids"][:, 0].contiguous() if case["alpha"] else None
        # the mean over the rows that count; one in eight is padding
        keep = (rand.whole(8, rows) > 0).float()
        keep[0] = 1.0
        s["weights"] = keep / keep.sum()
        s["loss"] = torch.zeros((rows,), device=DEVICE)
        s["delta"] = torch.zeros((rows, ld), device=DEVICE)
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------------------
def _cut(a, block_rows):
    """[rows, cols] padded with zeros to whole blocks, as [row blocks, block_rows, column blocks, 128]."""
    rows, cols = a.shape
    full = a.new_zeros((_blocks(rows, block_rows) * block_rows, _blocks(cols) * BLOCK))
    full[:rows, :cols] = a
    return full.view(-1, block_rows, _blocks(cols), BLOCK)


def _plain_quantize(a, form, block_rows, pow2):
    _, kind, largest, _, _ = FORMATS[form]
    cut = _cut(a, block_rows)
    peak = torch.clamp(cut.abs().amax((1, 3), keepdim=True), min=SMALLEST)
    whole = torch.full_like(peak, largest)
    scale, factor = torch.div(peak, whole), torch.div(whole, peak)
    if pow2:
        part, power = torch.frexp(peak)                    # peak = part 2^power, 1/2 <= part < 1
        most, least = math.frexp(largest)
        power = power - least + (part > most).int()
        scale, factor = torch.ldexp(torch.ones_like(peak), power), torch.ldexp(torch.ones_like(peak), -power)
    q = (cut * factor).view(cut.shape[0] * block_rows, -1)[:a.shape[0], :a.shape[1]].to(kind)
    return q, scale[:, 0, :, 0].t().contiguous()


def _plain_values(e):
    """What the 8-bit matrix stands for."""
    scale = e.scale.t().repeat_interleave(e.block_rows, 0)[:e.rows].repeat_interleave(BLOCK, 1)[:, :e.cols]
    return e.q.float() * scale


def _plain_product(a, b):
    return _plain_values(a) @ _plain_values(b).t()


class _Values:
    """A freshly quantised matrix with the fields of _Eight."""

    def __init__(self, a, form, block_rows):
        self.rows, self.cols, self.block_rows = a.shape[0], a.shape[1], block_rows
        self.q, self.scale = _plain_quantize(a, form, block_rows, True)


def _plain_norm(x, layer, eps):
    centred = x - x.mean(1, keepdim=True) if layer else x
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + eps)
    return centred * rstd, rstd


def _plain_norm_back(d, n, rstd, layer):
    back = d - n * (d * n).mean(1, keepdim=True)
    return rstd * (back - d.mean(1, keepdim=True) if layer else back)


def _plain_norm_residual(s, c):
    layer, eps = c["kind"] == "layer", s["eps"]
    gate = 1.0 if s["gate"] is None else s["gate"].repeat_interleave(c["rows"], 0)
    n1, rstd1 = _plain_norm(s["f"], layer, eps) if c["post"] else (s["f"], None)
    z = n1 if s["g1"] is None else n1 * s["g1"]
    z = z if s["b1"] is None else z + s["b1"]
    r_out = s["res_scale"] * s["r"] + gate * z
    n2, rstd2 = _plain_norm(r_out, layer, eps)
    h = n2 * s["g2"]
    out = {"r_out": r_out, "h": h if s["b2"] is None else h + s["b2"]}
    if c["train"]:
        dh = s["dh"]
        u = s["dr_out"] + _plain_norm_back(dh * s["g2"], n2, rstd2, layer)
        dz = gate * u
        dn = dz if s["g1"] is None else dz * s["g1"]
        out.update(dr=s["res_scale"] * u, df=_plain_norm_back(dn, n1, rstd1, layer) if c["post"] else dn, dg2=(dh * n2).sum(0))
        if s["b2"] is not None:
            out["db2"] = dh.sum(0)
        if s["g1"] is not None:
            out["dg1"] = (dz * n1).sum(0)
        if s["b1"] is not None:
            out["db1"] = dz.sum(0)
        if s["gate"] is not None:
            out["dgate"] = (u * z).view(c["groups"], c["rows"], -1).sum(1)
    return out


def _plain_softmax(x):
    """Largest value, exp(x - largest) and the sum of those, along the rows."""
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    return top, e, e.sum(1, keepdim=True)


def _plain_distill(s, c):
    cols, t, alpha = c["cols"], c["temperature"], c["alpha"]
    x, at, w = s["logits"][:, :cols], s["ids"].long(), s["weights"][:, None]
    top, e, total = _plain_softmax(x / t)
    q, log_q = e / total, (x.gather(1, at) / t - top) - torch.log(total)
    if s["teacher_lse"] is None:
        t_top, te, tt = _plain_softmax(s["teacher"] / t)
        p, log_p = te / tt, (s["teacher"] / t - t_top) - torch.log(tt)
        kl = (p * (log_p - log_q)).sum(1, keepdim=True)
        slope = q.scatter_add(1, at, -p)
    else:
        log_p = s["teacher"].double() / t - s["teacher_lse"].double()[:, None]
        p, log_p = torch.exp(log_p), log_p
        rest = torch.clamp(1.0 - p.sum(1, keepdim=True), min=0.0).float()
        p, log_p = p.float(), log_p.float()
        others = e.scatter(1, at, 0.0)
        q_rest = others.sum(1, keepdim=True) / total
        kl = (p * (log_p - log_q)).sum(1, keepdim=True) + torch.where(rest > 0, rest * torch.log(rest / q_rest), torch.zeros_like(rest))
        slope = (q - others / total * (rest / q_rest)).scatter_add(1, at, -p)
    loss, delta = (1 - alpha) * t * t * kl, (1 - alpha) * t * slope
    if alpha:
        label = s["labels"].long()[:, None]
        top1, e1, total1 = _plain_softmax(x)
        loss = loss + alpha * (torch.log(total1) - (x.gather(1, label) - top1))
        delta = delta + alpha * (e1 / total1).scatter_add(1, label, torch.full_like(total1, -1.0))
    return {"loss": (w * loss)[:, 0], "delta": w * delta}


def _plain(s):
    c = s["case"]
    if c["op"] == "fp8_product":
        return {"c": _plain_product(s["a"], s["b"])}
    if c["op"] == "fp8_quantize":
        q, scale = _plain_quantize(s["a"], c["format"], c["block_rows"], c["pow2"])
        qt, scale_t = _plain_quantize(s["a"].t(), c["format"], c["block_rows"], c["pow2"])
        return {"q": q, "scale": scale, "qt": qt, "scale_t": scale_t}
    if c["op"] == "fp8_dense":
        x, w, dy, form = s["x"], s["w"], s["dy"], c["format"]
        return {"y": _plain_product(_Values(x, "e4m3", 1), _Values(w, "e4m3", 128)),
                "dx": _plain_product(_Values(dy, form, 1), _Values(w.t(), "e4m3", 128)),
                "dw": _plain_product(_Values(dy.t(), form, 1), _Values(x.t(), "e4m3", 1))}
    return _plain_norm_residual(s, c) if c["op"] == "norm" else _plain_distill(s, c)


# ---- the framework's calls -----------------------------------------------------------------------------------------------------
def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_quantize(L, a, q, qt, pow2):
    L.call("fp8_quantize", DEV, a.data_ptr(), a.shape[0], a.shape[1], FORMATS[q.form][0], q.block_rows, int(pow2), q.store.data_ptr(), q.store.shape[1],
           q.scale.data_ptr(), qt.store.data_ptr(), qt.store.shape[1], qt.scale.data_ptr())


def _own_product(L, a, b, c):
    L.call("fp8_mult2d", DEV, *a.args(), *b.args(), c.data_ptr(), 0, a.rows, b.rows, a.cols)


def _own(s):
    from eddl_b200 import capi
    L, c = capi.lib(), s["case"]
    if c["op"] == "fp8_product":
        _own_product(L, s["a"], s["b"], s["c"])
        return {"c": s["c"]}
    if c["op"] == "fp8_quantize":
        _own_quantize(L, s["a"], s["q"], s["qt"], c["pow2"])
        return {"q": s["q"].q, "scale": s["q"].scale, "qt": s["qt"].q, "scale_t": s["qt"].scale}
    if c["op"] == "fp8_dense":
        _own_quantize(L, s["x"], s["xq"], s["xt"], True)
        _own_quantize(L, s["w"], s["wq"], s["wt"], True)
        _own_product(L, s["xq"], s["wq"], s["y"])
        _own_quantize(L, s["dy"], s["dq"], s["dt"], True)
        _own_product(L, s["dq"], s["wt"], s["dx"])
        _own_product(L, s["dt"], s["xt"], s["dw"])
        return {"y": s["y"], "dx": s["dx"], "dw": s["dw"]}
    if c["op"] == "norm":
        p = {k: _ptr(v) for k, v in s.items() if v is None or isinstance(v, torch.Tensor)}
        shape = (int(c["kind"] == "layer"), c["post"], c["groups"], c["rows"], c["cols"])
        L.call("norm_residual_fwd", DEV, *shape, p["f"], p["r"], p["gate"], p["g1"], p["b1"], s["res_scale"], p["g2"], p["b2"], s["eps"], p["r_out"], p["h"], p["stats"])
        if not c["train"]:
            return {"r_out": s["r_out"], "h": s["h"]}
        L.call("norm_residual_bwd", DEV, *shape, p["dh"], p["dr_out"], p["f"], p["r_out"], p["gate"], p["g1"], p["b1"], s["res_scale"], p["g2"], p["stats"],
               p["df"], p["dr"], 0, p["dgate"], p["dg1"], p["db1"], p["dg2"], p["db2"], 0)
        return {k: s[k] for k in ("r_out", "h", "df", "dr", "dgate", "dg1", "db1", "dg2", "db2") if s[k] is not None}
    L.call("distill", DEV, _ptr(s["logits"]), _ptr(s["ids"]), _ptr(s["teacher"]), _ptr(s["teacher_lse"]), _ptr(s["labels"]), _ptr(s["weights"]),
           c["rows"], c["cols"], c["cols"] + c["pad"], c["k"], c["temperature"], c["alpha"], _ptr(s["loss"]), _ptr(s["delta"]))
    return {"loss": s["loss"], "delta": s["delta"][:, :c["cols"]]}


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definition, in 64 bits --------------------------------------------------------------------------------------------------
def _exact_quantize(a, form, block_rows, pow2):
    """[rows, cols] in 64 bits: the 8-bit values, and the scales as [column block, row block]."""
    _, _, largest, bits, least = FORMATS[form]
    rows, cols = a.shape
    peak = torch.nn.functional.max_pool2d(a.abs()[None], (block_rows, BLOCK), ceil_mode=True)[0].clamp(min=SMALLEST)
    each = peak.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    scale, factor = peak / largest, largest / each
    if pow2:
        scale, factor = torch.exp2(torch.ceil(torch.log2(scale))), torch.exp2(-torch.ceil(torch.log2(each / largest)))
    x = a * factor
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** least))) - bits)
    return (torch.round(x / step) * step).clamp(-largest, largest), scale.t()


def _exact_product(qa, sa, block_a, qb, sb, block_b):
    c = 0.0
    for b in range(sa.shape[0]):
        at = slice(b * BLOCK, (b + 1) * BLOCK)
        left = sa[b].repeat_interleave(block_a)[:qa.shape[0]]
        right = sb[b].repeat_interleave(block_b)[:qb.shape[0]]
        c = c + (qa[:, at] * left[:, None]) @ (qb[:, at] * right[:, None]).t()
    return c


def _exact_norm(x, kind, eps):
    if kind == "layer":
        return torch.nn.functional.layer_norm(x, x.shape[1:], eps=eps)
    return x * torch.rsqrt(x.pow(2).mean(1, keepdim=True) + eps)


def _exact_distill(s, c):
    t, alpha, at = c["temperature"], c["alpha"], s["ids"].long()
    x = s["logits"][:, :c["cols"]].double().requires_grad_()
    log_q = torch.log_softmax(x / t, 1)
    picked = log_q.gather(1, at)
    if c["tail"]:
        log_p = s["teacher"].double() / t - s["teacher_lse"].double()[:, None]
        p = log_p.exp()
        rest = (1.0 - p.sum(1)).clamp(min=0.0)
        outside = torch.logsumexp(log_q.scatter(1, at, -math.inf), 1)
        kl = (p * (log_p - picked)).sum(1) + torch.xlogy(rest, rest) - rest * outside
    else:
        log_p = torch.log_softmax(s["teacher"].double() / t, 1)
        kl = (log_p.exp() * (log_p - picked)).sum(1)
    loss = (1 - alpha) * t * t * kl
    if alpha:
        loss = loss + alpha * torch.nn.functional.cross_entropy(x, s["labels"].long(), reduction="none")
    loss = loss * s["weights"].double()
    return {"loss": loss.detach(), "delta": torch.autograd.grad(loss.sum(), x)[0]}


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "fp8_product":
        a, b = s["a"], s["b"]
        return {"c": _exact_product(a.q.double(), a.scale.double(), 1, b.q.double(), b.scale.double(), b.block_rows)}
    if op == "fp8_quantize":
        a = s["a"].double()
        q, scale = _exact_quantize(a, case["format"], case["block_rows"], case["pow2"])
        qt, scale_t = _exact_quantize(a.t().contiguous(), case["format"], case["block_rows"], case["pow2"])
        return {"q": q, "scale": scale, "qt": qt, "scale_t": scale_t}
    if op == "fp8_dense":
        x, w, dy, form = s["x"].double(), s["w"].double(), s["dy"].double(), case["format"]

        def product(a, form_a, b, block_b):
            return _exact_product(*_exact_quantize(a.contiguous(), form_a, 1, True), 1, *_exact_quantize(b.contiguous(), "e4m3", block_b, True), block_b)
        return {"y": product(x, "e4m3", w, 128), "dx": product(dy, form, w.t(), 128), "dw": product(dy.t(), form, x.t(), 1)}
    if op == "distill":
        return _exact_distill(s, case)
    v = {k: s[k].double().requires_grad_() for k in ("f", "r", "gate", "g1", "b1", "g2", "b2") if s[k] is not None}
    z = _exact_norm(v["f"], case["kind"], s["eps"]) if case["post"] else v["f"]
    z = z * v["g1"] if "g1" in v else z
    z = z + v["b1"] if "b1" in v else z
    r_out = s["res_scale"] * v["r"] + (z.view(case["groups"], case["rows"], -1) * v["gate"][:, None] if "gate" in v else z).view_as(z)
    h = _exact_norm(r_out, case["kind"], s["eps"]) * v["g2"]
    h = h + v["b2"] if "b2" in v else h
    out = {"r_out": r_out.detach(), "h": h.detach()}
    if case["train"]:
        names = list(v)
        grads = torch.autograd.grad((r_out, h), [v[k] for k in names], (s["dr_out"].double(), s["dh"].double()))
        out.update({"d" + k: g for k, g in zip(names, grads)})
    return out


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "fp8_product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": float(m * k + n * k + 4 * m * n), "flops": 2.0 * m * n * k}
    if op == "fp8_quantize":
        # fp32 in, one byte out for each of the two directions
        size = case["rows"] * case["cols"]
        return {"bytes": 6.0 * size, "flops": 4.0 * size}
    if op == "fp8_dense":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 8.0 * (m * k + n * k + m * n), "flops": 6.0 * m * n * k}
    if op == "norm":
        # f, r read, r_out, h written; training: dh, dr_out read and df, dr written as well (f and r_out need not leave the chip's
        # reach between the two passes of this case, so they are counted once)
        size = case["groups"] * case["rows"] * case["cols"]
        return {"bytes": (32.0 if case["train"] else 16.0) * size, "flops": (40.0 if case["train"] else 14.0) * size}
    size = case["rows"] * case["cols"]
    return {"bytes": 8.0 * size + 8.0 * case["rows"] * case["k"], "flops": 12.0 * size}
