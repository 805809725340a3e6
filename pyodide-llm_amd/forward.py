"""A ragged batch of tokens through the layers of a loaded checkpoint: a serving step, prompts and single tokens together,
over a paged cache.

A layer is eight calls of the library and two of torch's element-wise operations (the rotation of queries and keys, the
feed-forward's gate), the residual stream in float32 and every product's activations quantized on their way:

    hq_norm_ready_ex    x += what the layer before gave; norm; readied for q, k and v
    hq_phase            q, k, v
    (rotation)
    hq_cache_write_ex   the new keys and values, quantized into their pages
    hq_attention_ex     over all pages of each sequence
    hq_matmuls          the attention's product
    hq_norm_ready_ex    x += it; norm; readied for the gate and the up product
    hq_phase            both
    (gate)
    hq_matmuls          the down product

The forward pass of the reference (src/runtime/forward/engine.ts) takes one sequence and a cache as long as the model's
sequence; its products are these, the operators between them are its own.
"""
from . import check, jobs, library
from .cache import FORMS, READY, READY_BYTES, Batch, Cache, shapes


class Forward:
    """The buffers of steps of up to `tokens` tokens of `sequences` sequences over `pages` pages of `page` positions a layer;
    a sequence has up to `width` pages."""

    def __init__(self, ck, tokens, sequences, pages, width, page=64, form="int8", eps=1e-5, theta=10000.0):
        torch, s, device = ck.torch, ck.shape, ck.device
        self.ck, self.torch, self.lib, self.eps = ck, torch, library(), eps
        self.tokens, self.sequences, self.pages, self.width, self.page, self.form = (tokens, sequences, pages, width, page,
                                                                                     form)
        self.ready = READY["planes" if ck.dtype in ("ternary", "binary") else "biased" if ck.relaxed else "plain"]
        scales = READY_BYTES[{v: k for k, v in READY.items()}[self.ready]]
        self.frames = {n: -(-(n + scales(n)) // 256) * 256 for n in (s.dim, s.hidden_dim, s.heads * s.head_size)}
        self.norms = {name: torch.from_numpy(v).to(device) for name, v in ck.vectors.items() if name.startswith("rms_")}

        def floats(*shape):
            return torch.empty(shape, dtype=torch.float32, device=device)

        self.q, self.att = floats(tokens, s.heads, s.head_size), floats(tokens, s.heads, s.head_size)
        self.k, self.v = floats(tokens, s.kv_heads, s.head_size), floats(tokens, s.kv_heads, s.head_size)
        self.given, self.y = floats(tokens, s.dim), floats(tokens, s.dim)
        self.gate, self.up = floats(tokens, s.hidden_dim), floats(tokens, s.hidden_dim)
        self.xq = torch.empty(tokens * max(self.frames.values()), dtype=torch.uint8, device=device)
        # a layer's cache is (k, v, ks, vs); no value is needed to start with
        k, v, scale, _ = shapes(form, pages, page, s.kv_heads, s.head_size)
        element = torch.int8 if form == "int8" else torch.float16
        self.held = [(torch.empty(k, dtype=element, device=device), torch.empty(v, dtype=element, device=device),
                      floats(*scale), floats(*scale)) for _ in range(s.layers)]
        self.caches = [Cache(*(t.data_ptr() for t in held), FORMS[form], pages, page, s.kv_heads, s.head_size)
                       for held in self.held]
        self.work = torch.empty(0, dtype=torch.uint8, device=device)
        half = torch.arange(0, s.head_size, 2, device=device, dtype=torch.float64) / s.head_size
        angles = torch.arange(width * page, device=device, dtype=torch.float64)[:, None] * theta ** -half
        self.turn = torch.polar(torch.ones_like(angles), angles).to(torch.complex64)

    def products(self, names, layer, x, outs, count, stream, readied):
        """outs[i] = names[i]'s product of the readied activations, or of x's"""
        n = self.ck.matrices[names[0]].n
        frame, xq = self.frames[n], self.xq.data_ptr()
        table = []
        for name, out in zip(names, outs):
            m = self.ck.matrices[name]
            table.append(m.job(layer, out.data_ptr(), xq, xq + n, count, 4 * m.rows, frame))
        check(jobs.phase(self.lib, table, stream) if readied else jobs.matmuls(self.lib, x.data_ptr(), 4 * n, table, stream))

    def norm(self, x, given, weight, count, stream, y=None):
        """x += given; y = its norm, or the next products' activations"""
        n, s = x.shape[1], stream.cuda_stream
        xq = 0 if y is not None else self.xq.data_ptr()
        check(self.lib.hq_norm_ready_ex(xq, xq and xq + n, 0 if y is None else y.data_ptr(), x.data_ptr(), x.data_ptr(),
                                        0 if given is None else given.data_ptr(), weight.data_ptr(), n, self.eps, self.ready,
                                        count, self.frames[n], 4 * n, 4 * n, 4 * n, s))

    def rotate(self, t, at):
        """pairs of neighbouring values turned by their position's angles"""
        pairs = self.torch.view_as_complex(t.view(*t.shape[:-1], -1, 2))
        pairs.mul_(self.turn[at][:, None, :])

    def step(self, x, starts, lengths, table, longest=0):
        """x: the new tokens' embeddings (float32, on the device), which become the residual stream; starts, lengths and
        table: hq_batch's, int32 on the device, lengths with the new tokens among them; longest: the most new tokens that a
        sequence has (0: not known, which makes a step of single tokens slower).  Returns the final norm of every new token's row
        (a buffer of this object's)."""
        torch, lib, ck, s = self.torch, self.lib, self.ck, self.ck.shape
        count, sequences = x.shape[0], lengths.shape[0]
        if not (x.dim() == 2 and 0 < count <= self.tokens and 0 < sequences <= self.sequences and x.shape[1] == s.dim
                and tuple(table.shape) == (sequences, self.width) and tuple(starts.shape) == (sequences + 1,)
                and lengths.dim() == 1):
            raise ValueError(f"refused: {tuple(x.shape)} embeddings, a table of {tuple(table.shape)}, {tuple(starts.shape)} starts "
                             f"and {tuple(lengths.shape)} lengths for steps of {self.tokens} tokens, {self.sequences} sequences "
                             f"of {self.width} pages")
        # the calls take addresses: what lies there has to be what they read (and write: x is the residual stream)
        for name, t, kind in (("x", x, torch.float32), ("starts", starts, torch.int32), ("lengths", lengths, torch.int32),
                              ("table", table, torch.int32)):
            if t.dtype != kind or not t.is_contiguous() or t.device != self.y.device:
                raise ValueError(f"refused: {name} is {t.dtype} on {t.device}, not {kind} on {self.y.device} in one piece")
        stream = torch.cuda.current_stream()
        batch = Batch(starts.data_ptr(), lengths.data_ptr(), table.data_ptr(), sequences, count, longest, self.width)
        needed = lib.hq_attention_work_bytes(self.caches[0], batch, s.heads)
        if needed < 0:
            check(needed)
        if self.work.numel() < needed:
            self.work = torch.empty(needed, dtype=torch.uint8, device=x.device)
        # a token's position: its place before its sequence's end
        rows = torch.arange(count, device=x.device, dtype=torch.int32)
        mine = (torch.searchsorted(starts, rows, right=True) - 1).clamp_(0, sequences - 1)
        at = (lengths[mine] - (starts[mine + 1] - rows)).clamp_(0, self.turn.shape[0] - 1).long()
        q, k, v, att = self.q[:count], self.k[:count], self.v[:count], self.att[:count]
        gate, up, given = self.gate[:count], self.up[:count], self.given[:count]
        wide, narrow = 4 * s.heads * s.head_size, 4 * s.kv_heads * s.head_size
        for layer, cache in enumerate(self.caches):
            self.norm(x, given if layer else None, self.norms["rms_att_weight"][layer], count, stream)
            self.products(("wq", "wk", "wv"), layer, None, (q, k, v), count, stream, True)
            self.rotate(q, at)
            self.rotate(k, at)
            check(lib.hq_cache_write_ex(cache, batch, k.data_ptr(), v.data_ptr(), narrow, narrow, stream.cuda_stream))
            check(lib.hq_attention_ex(att.data_ptr(), q.data_ptr(), s.heads, wide, wide, cache, batch, s.head_size ** -0.5, 0,
                                      0.0, self.work.data_ptr(), self.work.numel(), stream.cuda_stream))
            self.products(("wo",), layer, att, (given,), count, stream, False)
            self.norm(x, given, self.norms["rms_ffn_weight"][layer], count, stream)
            self.products(("w1", "w3"), layer, None, (gate, up), count, stream, True)
            torch.nn.functional.silu(gate, inplace=True).mul_(up)
            self.products(("w2",), layer, gate, (given,), count, stream, False)
        y = self.y[:count]
        self.norm(x, given, self.norms["rms_final_weight"], count, stream, y)
        return y
