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

A step may carry low-rank adapters (hq_adapters_ex after the products that they stand beside), and embed() and logits() are what
comes before and after the layers (serve.py runs them all).

The forward pass of the reference (src/runtime/forward/engine.ts) takes one sequence and a cache as long as the model's
sequence; its products are these, the operators between them are its own.
"""
import functools

from . import HQ_PACK, check, jobs, library
from .adapters import Target
from .cache import FORMS, READY, READY_BYTES, Batch, Cache, shapes


def on_its_device(method):
    """`method` with the device of its object's buffers as the current one, on which the library's calls run"""
    @functools.wraps(method)
    def run(self, *args, **kwargs):
        if self.device.type != "cuda":  # (nothing runs on the host's memory)
            return method(self, *args, **kwargs)
        with self.torch.cuda.device(self.device):
            return method(self, *args, **kwargs)
    return run


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
        self.device = self.y.device
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
        self.captured = False  # (whether a captured step uses this workspace: it is kept then)
        self.older = []  # (such workspaces that were too small for a later step)
        self.normed = None  # (a norm's values beside the readied ones: where adapters read them)
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

    def norm(self, x, given, weight, count, stream, y=None, both=False):
        """x += given; y = its norm, or (with `both`: and) the next products' activations"""
        n, s = x.shape[1], stream.cuda_stream
        xq = 0 if y is not None and not both else self.xq.data_ptr()
        check(self.lib.hq_norm_ready_ex(xq, xq and xq + n, 0 if y is None else y.data_ptr(), x.data_ptr(), x.data_ptr(),
                                        0 if given is None else given.data_ptr(), weight.data_ptr(), n, self.eps, self.ready,
                                        count, self.frames[n], 4 * n, 4 * n, 4 * n, s))

    def adapt(self, adapters, names, layer, x, outs, batch, which, stream):
        """outs[i] += names[i]'s adapters of x's rows, each sequence's its own"""
        pairs = [(name, out) for name, out in zip(names, outs) if name in adapters.factors]
        if not pairs:
            return
        targets = (Target * len(pairs))(*(adapters.target(name, layer, out, 4 * self.ck.matrices[name].rows)
                                          for name, out in pairs))
        n = self.ck.matrices[names[0]].n
        check(self.lib.hq_adapters_ex(targets, len(pairs), x.data_ptr(), 4 * n, n, adapters.rank, adapters.count, adapters.form,
                                      0 if adapters.scales is None else adapters.scales.data_ptr(), which.data_ptr(), batch,
                                      self.work.data_ptr(), self.work.numel(), stream.cuda_stream))

    def adapters_fit(self, adapters, count):
        """the bytes of workspace of a step of `count` tokens with these adapters"""
        ck = self.ck
        for name, (a, b) in adapters.factors.items():
            m = ck.matrices.get(name) if name in ("wq", "wk", "wv", "wo", "w1", "w3", "w2") else None
            if m is None or a.shape[0] != m.layers or a.shape[3] != m.n or b.shape[2] != m.rows or a.device != self.y.device:
                raise ValueError(f"refused: {name}'s factors of {tuple(a.shape)} and {tuple(b.shape)} on {a.device}")
        return self.lib.hq_adapters_work_bytes(3, adapters.rank, count)

    @on_its_device
    def embed(self, ids, x, scale=1.0):
        """x (float32 rows) = the embeddings of ids (int32), both on the device; an id that is none gives zeros"""
        m, s = self.ck.matrices["token_embedding_table"], self.ck.shape
        for name, t, kind, shape in (("ids", ids, "torch.int32", (x.shape[0],)), ("x", x, "torch.float32", (x.shape[0], s.dim))):
            if str(t.dtype) != kind or tuple(t.shape) != shape or not t.is_contiguous() or t.device != self.y.device:
                raise ValueError(f"refused: {name} is {tuple(t.shape)} of {t.dtype} on {t.device}, not {shape} of {kind} on "
                                 f"{self.y.device} in one piece")
        check(self.lib.hq_embed_ex(x.data_ptr(), ids.data_ptr(), m.values, m.scales, HQ_PACK[m.kind], s.vocab, s.dim, scale,
                                   x.shape[0], 4 * s.dim, self.torch.cuda.current_stream().cuda_stream))

    @on_its_device
    def logits(self, y, out):
        """out[i] = the classifier's logits of y[i], a final norm's row whose outlier channels are set to 0 on the way, as
        Checkpoint.classify's are: one product for all rows, the channels a row after another"""
        ck, s, count = self.ck, self.ck.shape, y.shape[0]
        for name, t, width in (("y", y, s.dim), ("out", out, s.vocab)):
            if (str(t.dtype) != "torch.float32" or tuple(t.shape) != (count, width) or not t.is_contiguous()
                    or t.device != self.y.device or count > self.tokens):
                raise ValueError(f"refused: {name} is {tuple(t.shape)} of {t.dtype} on {t.device}, for up to {self.tokens} rows of "
                                 f"{width} float32 on {self.y.device}")
        if count == 0:
            return
        stream = self.torch.cuda.current_stream()
        channels = len(ck.channels)
        if channels:
            picked = self.torch.empty(count, channels, dtype=self.torch.float32, device=y.device)
            for i in range(count):
                check(self.lib.hq_take_channels_ex(picked[i].data_ptr(), y[i].data_ptr(), ck._channels, channels,
                                                   stream.cuda_stream))
        m, frame, xq = ck.classifier, self.frames[s.dim], self.xq.data_ptr()
        check(jobs.matmuls(self.lib, y.data_ptr(), 4 * s.dim,
                           [m.job(0, out.data_ptr(), xq, xq + s.dim, count, 4 * s.vocab, frame)], stream))
        for i in range(count if channels else 0):
            check(self.lib.hq_add_columns_ex(out[i].data_ptr(), ck.columns.data_ptr(), picked[i].data_ptr(), channels, s.vocab,
                                             stream.cuda_stream))

    def rotate(self, t, at):
        """pairs of neighbouring values turned by their position's angles"""
        pairs = self.torch.view_as_complex(t.view(*t.shape[:-1], -1, 2))
        pairs.mul_(self.turn[at][:, None, :])

    @on_its_device
    def step(self, x, starts, lengths, table, longest=0, at=None, adapters=None, which=None):
        """x: the new tokens' embeddings (float32, on the device), which become the residual stream; starts, lengths and
        table: hq_batch's, int32 on the device, lengths with the new tokens among them; longest: the most new tokens that a
        sequence has (0: not known, which makes a step of single tokens slower); at: each row's position (int32, as
        hq_batch_plan_ex gives it; None: worked out here); adapters (an Adapters) and which (int32): each sequence's, none where
        it is no adapter's number.  Returns the final norm of every new token's row
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
                              ("table", table, torch.int32), ("at", at, torch.int32), ("which", which, torch.int32)):
            if t is None and name in ("at", "which"):
                continue
            if t.dtype != kind or not t.is_contiguous() or t.device != self.y.device:
                raise ValueError(f"refused: {name} is {t.dtype} on {t.device}, not {kind} on {self.y.device} in one piece")
        if ((adapters is None) != (which is None) or (at is not None and tuple(at.shape) != (count,))
                or (which is not None and tuple(which.shape) != (sequences,))):
            raise ValueError(f"refused: positions and adapters for {count} tokens of {sequences} sequences: at "
                             f"{at if at is None else tuple(at.shape)}, which {which if which is None else tuple(which.shape)}, "
                             f"adapters {adapters}")
        extra = 0 if adapters is None else self.adapters_fit(adapters, count)
        if extra < 0:
            check(extra)
        stream = torch.cuda.current_stream()
        batch = Batch(starts.data_ptr(), lengths.data_ptr(), table.data_ptr(), sequences, count, longest, self.width)
        needed = lib.hq_attention_work_bytes(self.caches[0], batch, s.heads)
        if needed < 0:
            check(needed)
        needed = max(needed, extra)
        # (what is made while a step is captured is the graph's memory, and stays as long as this object)
        capturing = torch.cuda.is_current_stream_capturing()
        if self.work.numel() < needed:
            if self.captured or capturing:
                self.older.append(self.work)
            else:
                self.work.record_stream(stream)  # (it may be another stream's)
            self.work, self.captured = torch.empty(needed, dtype=torch.uint8, device=x.device), False
        self.captured = self.captured or capturing
        if at is None:
            # a token's position: its place before its sequence's end
            rows = torch.arange(count, device=x.device, dtype=torch.int32)
            mine = (torch.searchsorted(starts, rows, right=True) - 1).clamp_(0, sequences - 1)
            at = lengths[mine] - (starts[mine + 1] - rows)
        at = at.clamp(0, self.turn.shape[0] - 1).long()
        normed, both = None, {}
        if adapters is not None:
            if self.normed is None:
                self.normed = torch.empty_like(self.y)
            normed = self.normed[:count]
            both = dict(y=normed, both=True)

        def adapt(names, x, outs):
            if adapters is not None:
                self.adapt(adapters, names, layer, x, outs, batch, which, stream)

        q, k, v, att = self.q[:count], self.k[:count], self.v[:count], self.att[:count]
        gate, up, given = self.gate[:count], self.up[:count], self.given[:count]
        wide, narrow = 4 * s.heads * s.head_size, 4 * s.kv_heads * s.head_size
        for layer, cache in enumerate(self.caches):
            self.norm(x, given if layer else None, self.norms["rms_att_weight"][layer], count, stream, **both)
            self.products(("wq", "wk", "wv"), layer, None, (q, k, v), count, stream, True)
            adapt(("wq", "wk", "wv"), normed, (q, k, v))
            self.rotate(q, at)
            self.rotate(k, at)
            check(lib.hq_cache_write_ex(cache, batch, k.data_ptr(), v.data_ptr(), narrow, narrow, stream.cuda_stream))
            check(lib.hq_attention_ex(att.data_ptr(), q.data_ptr(), s.heads, wide, wide, cache, batch, s.head_size ** -0.5, 0,
                                      0.0, self.work.data_ptr(), self.work.numel(), stream.cuda_stream))
            self.products(("wo",), layer, att, (given,), count, stream, False)
            adapt(("wo",), att, (given,))
            self.norm(x, given, self.norms["rms_ffn_weight"][layer], count, stream, **both)
            self.products(("w1", "w3"), layer, None, (gate, up), count, stream, True)
            adapt(("w1", "w3"), normed, (gate, up))
            torch.nn.functional.silu(gate, inplace=True).mul_(up)
            self.products(("w2",), layer, gate, (given,), count, stream, False)
            adapt(("w2",), gate, (given,))
        y = self.y[:count]
        self.norm(x, given, self.norms["rms_final_weight"], count, stream, y)
        return y
