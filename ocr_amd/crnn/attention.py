"""A decoder's cross-attention layer over the recogniser's line states.

The recogniser answers a line timestep by timestep (arg-max and CTC).  A decoder that writes a line's text itself, or
queries that look for a field over all lines of a page, read many states at once: ``CRNN.line_states`` gives them,
``LineAttention.memory`` turns them into keys and values once, and each call of the layer attends to those.

    crnn = CRNN(...); crnn.load_weights(path)
    layer = LineAttention(crnn, weights, heads=8)
    states, lengths = crnn.line_states(lines)          # uint8 [n, 32, w] on the device
    memory = layer.memory(states, lengths)             # once per batch of lines; or page_memory: all lines as one memory
    y = layer(x, memory)                               # x [n, t, dim]: one row a step (t = 1) or a whole text
"""
import collections

LineMemory = collections.namedtuple("LineMemory", ["k", "v", "lengths", "mask"])


class LineAttention(object):
    """y = t + out(attention(q(norm(t)), k, v)), t = x (+ residual); operators of ``CRNN`` (seq_ops.py) throughout.

    weights: "norm.weight" float32 [dim]; "q.weight" [heads * d, dim], "kv.weight" [2 * kv_heads * d, 512] (keys before
    values), "out.weight" [dim, heads * d], all float32 or all bfloat16, tensors on the handle's device; optional float32
    biases "q.bias", "kv.bias", "out.bias".  "q.weight" may be float8_e4m3fn with a float32 "q.scale" [heads * d] where the
    others are bfloat16: the norm then leaves 8-bit rows for it.  d is 1 .. 128; heads of whole 16-byte chunks (8 bfloat16, 4
    float32 values) are several times faster."""

    def __init__(self, crnn, weights, heads, kv_heads=None, eps=1e-6):
        import torch
        self.crnn, self.heads, self.kv_heads, self.eps = crnn, heads, kv_heads or heads, eps
        self.w = {k: v.detach() for k, v in weights.items()}
        known = {"norm.weight", "q.weight", "q.bias", "q.scale", "kv.weight", "kv.bias", "out.weight", "out.bias"}
        missing, extra = {"norm.weight", "q.weight", "kv.weight", "out.weight"} - set(self.w), set(self.w) - known
        if missing or extra:
            raise ValueError("LineAttention: missing weights %s, unknown weights %s" % (sorted(missing), sorted(extra)))
        self.dtype = self.w["kv.weight"].dtype
        q = self.w["q.weight"]
        self.q8 = q.dtype is torch.float8_e4m3fn
        if self.dtype not in (torch.float32, torch.bfloat16) or self.w["out.weight"].dtype is not self.dtype or \
                (q.dtype is not self.dtype and not (self.q8 and self.dtype is torch.bfloat16)) or self.q8 != ("q.scale" in self.w):
            raise ValueError("LineAttention: the weights have to be all float32 or all bfloat16 (q.weight: or float8_e4m3fn with q.scale)")
        if q.dim() != 2 or heads < 1 or self.kv_heads < 1 or heads % self.kv_heads or q.shape[0] % heads:
            raise ValueError("LineAttention: q.weight %s does not fit %d heads over %d" % (tuple(q.shape), heads, self.kv_heads))
        self.d, self.dim = q.shape[0] // heads, q.shape[1]
        if not 1 <= self.d <= 128:
            raise ValueError("LineAttention: q.weight %s gives heads of %d, 1 .. 128 are possible" % (tuple(q.shape), self.d))
        for name, shape in (("kv.weight", (2 * self.kv_heads * self.d, 512)), ("out.weight", (self.dim, heads * self.d))):
            if tuple(self.w[name].shape) != shape:
                raise ValueError("LineAttention: %s has to be %s, got %s" % (name, shape, tuple(self.w[name].shape)))
        for name, size in (("norm.weight", self.dim), ("q.bias", heads * self.d), ("q.scale", heads * self.d), ("kv.bias", 2 * self.kv_heads * self.d),
                           ("out.bias", self.dim)):
            t = self.w.get(name)
            if t is not None and (tuple(t.shape) != (size,) or t.dtype is not torch.float32):
                raise ValueError("LineAttention: %s has to be float32 [%d], got %s %s" % (name, size, t.dtype, tuple(t.shape)))

    def memory(self, states, lengths=None):
        """Keys and values of ``states`` [n, T, 512] (``CRNN.line_states``), a memory of its own for each line."""
        n, T, _ = states.shape
        kv = self.crnn.linear(states.to(self.dtype), self.w["kv.weight"], bias=self.w.get("kv.bias")).view(n, T, 2, self.kv_heads, self.d)
        return LineMemory(kv[:, :, 0], kv[:, :, 1], lengths, None)

    def page_memory(self, states, lengths=None):
        """The lines of one page as ONE memory [1, n T]: what is behind a line's end is masked out."""
        import torch
        n, T, _ = states.shape
        m = self.memory(states)
        mask = None
        if lengths is not None:
            mask = (torch.arange(T, device=states.device) < lengths[:, None]).view(1, n * T)
        return LineMemory(*(t.unflatten(0, (1, n)).flatten(1, 2) for t in m[:2]), None, mask)

    def __call__(self, x, memory, residual=None):
        """x, residual [n, t, dim] in the weights' type -> [n, t, dim]."""
        import torch
        c, w = self.crnn, self.w
        n, t, _ = x.shape
        y, scale, total = c.rms_norm(x, w["norm.weight"], residual=residual, eps=self.eps, out_dtype=torch.float8_e4m3fn if self.q8 else None)
        q = c.linear(y, w["q.weight"], bias=w.get("q.bias"), x_scale=scale, w_scale=w.get("q.scale")).view(n, t, self.heads, self.d)
        a = c.cross_attention(q, memory.k, memory.v, lengths=memory.lengths, mask=memory.mask).view(n, t, self.heads * self.d)
        return c.linear(a, w["out.weight"], bias=w.get("out.bias"), residual=x if total is None else total)
