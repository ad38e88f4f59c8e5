"""Workspaces that calls share: linears of several sizes on one stream, graphs whose stream
went on to larger calls, and paged forward passes on several streams and in graphs."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(cuda):
    import torch as _t
    return _t


@pytest.fixture(scope="module")
def lib(cuda):
    import dial_cuda
    return dial_cuda


@pytest.fixture(autouse=True)
def no_device_error(cuda):
    import dial_cuda
    yield
    assert dial_cuda.lib().dial_device_error(1) == 0, "a kernel reported an error"


def gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("qtype", ["Q4_0", "Q8_0"])
@pytest.mark.parametrize("K", [512, 1152, 2080])
@pytest.mark.parametrize("M", [1, 9])
def test_gguf_linears_of_several_sizes_on_one_stream(torch, lib, qtype, K, M):
    """A linear with few outputs between two calls of one with many: the same bits each time."""
    g = gen(torch, K + M)
    lins = [lib.GgufLinear.quantize(torch.randn((N, K), generator=g, device="cuda") * 0.05, getattr(lib, qtype))
            for N in (2048, 512, 1024, 16)]
    x = torch.randn((M, K), generator=g, device="cuda").half()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        want = [l.forward(x) for l in lins]
        for _ in range(3):
            for i in (0, 1, 3, 2, 0):
                got = lins[i].forward(x)
                side.synchronize()
                assert torch.equal(got, want[i]), i
    for l, y in zip(lins, want):
        ref = x.double() @ l.dequantize(torch.float32).double().T
        # the activations' Q8_0 rounding: half a step of absmax / 127 a value
        bound = (x.abs().amax(-1, keepdim=True).double() / 254 * 1.01) * l.dequantize(torch.float32).double().abs().sum(-1) + 2.0 ** -11 * ref.abs() + 1e-6
        assert torch.all((y.double() - ref).abs() <= bound)


# ------------------------------------------------------------------ a decoder over pages
CONFIGS = {
    "w8a16": dict(n_layers=2, hidden=512, intermediate=1024, n_heads=8, n_kv_heads=2, vocab=2048, act_dtype="bf16"),
    "q4_0": dict(n_layers=2, hidden=1152, intermediate=2304, n_heads=8, n_kv_heads=4, vocab=2048, qk_norm=False,
                 weight_format=2, head_format=8),  # Q4_0 layers, Q8_0 head
    "q8_0": dict(n_layers=2, hidden=1024, intermediate=1152, n_heads=4, n_kv_heads=4, vocab=999, weight_format=8, head_format=8),
}


class Paged:
    """A small decoder and one sequence's pages."""

    def __init__(self, torch, name, n_slots=1, max_seq=256):
        from dial_cuda import paged as P
        from dial_cuda.model import Decoder, ModelConfig
        self.torch, self.P, self.cfg = torch, P, ModelConfig(**CONFIGS[name])
        self.dec = Decoder(self.cfg, n_slots=n_slots, max_seq=max_seq)
        self.tables = P.rope_tables(max_seq, self.cfg.rope_theta)
        self.i32 = dict(dtype=torch.int32, device="cuda")

    def state(self, seed, quantized=False):
        """Caches of their own, filled by a first chunk of 40 tokens."""
        s = type("State", (), {})()
        s.caches = self.dec.stage.paged_caches(10, 16, quantized)
        s.table = self.torch.randperm(10, generator=gen(self.torch, seed), device="cuda").int().view(1, 10)
        s.ids = self.torch.randint(0, self.cfg.vocab, (120,), generator=gen(self.torch, seed + 1), **self.i32)
        self.chunk(s, 0, 40)
        return s

    def chunk(self, s, lo, hi, **kw):
        """A call over tokens lo .. hi, with tensors that stay."""
        i32, torch = self.i32, self.torch
        s.args = (s.ids[lo:hi].contiguous(), torch.arange(lo, hi, **i32),
                  self.P.PagedBatch(s.table, torch.tensor([hi], **i32), torch.tensor([0, hi - lo], **i32), max_q=hi - lo), s.caches)
        return self.call(s.args, **kw)

    def call(self, args, **kw):
        ids, pos, batch, caches = args
        return self.dec.forward_paged(ids, pos, batch, caches, self.tables, **kw)


@pytest.mark.parametrize("name", list(CONFIGS))
def test_forward_paged_agrees_with_the_slot_decoder(torch, lib, name):
    """A prompt, then four tokens at once and one.

    Both paths round every stage of a layer to the type: 12 roundings of u = eps / 2 at most a
    layer (norm, qkv, norm and turn in up to 4 steps, attention, o, sum, gate_up, swiglu, down),
    with embedding, last norm and logits 27 in two layers.  A rounding moves a vector by
    u / 3^.5 of its norm (uniform within half a step of at most u), the two paths' 54 add as
    independent ones: 18^.5 u of the logits' rms, and the largest of up to 2^17 logits is within
    4.8 of these: 20.4 u.  GGUF linears of up to 16 rows round their activations to Q8_0 as well,
    half a step of absmax / 127, where absmax is at most 3.5 times a block's rms on the average:
    0.8 % of it, by 2 x 9 linears and the same 4.8: 0.17 of the rms, for the calls of up to 16 tokens
    and, as attention averages the rows they left in the caches, for those behind them."""
    p = Paged(torch, name)
    s = p.state(5)
    st = p.dec.stage
    hidden = torch.empty((120, p.cfg.hidden), device="cuda", dtype=st.dt)
    for lo, hi in ((0, 40), (40, 44), (44, 45), (45, 100)):
        got, best = p.chunk(s, lo, hi)
        st.embed_tokens(s.ids[lo:hi].contiguous(), hidden[lo:hi])
        st.layers_forward(hidden[lo:hi], torch.arange(lo, hi, **p.i32), torch.zeros(hi - lo, **p.i32), hi)
        want = torch.empty((hi - lo, p.cfg.vocab), device="cuda", dtype=st.dt)
        st.head_forward(hidden[lo:hi], torch.empty(hi - lo, **p.i32), logits=want)
        bound = 20.4 * torch.finfo(st.dt).eps / 2 + (0.17 if name != "w8a16" and hi > 40 else 0.0)
        off, rms = float((got.float() - want.float()).abs().max()), float(want.float().square().mean().sqrt())
        assert off <= bound * rms, (lo, hi, off / rms)
        assert torch.equal(best.long(), got.float().argmax(-1))


@pytest.mark.parametrize("name", list(CONFIGS))
def test_forward_paged_on_two_streams_at_once(torch, lib, name):
    """Passes over caches of their own, on two streams: the bits of passes in turn."""
    p = Paged(torch, name)
    states = [p.state(b) for b in (1, 2)]
    want = [p.chunk(s, 40, 40 + n)[0] for s, n in zip(states, (3, 5))]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = []
    for _ in range(30):
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                got.append(p.call(s.args)[0])
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 2]), i


@pytest.mark.parametrize("name", list(CONFIGS))
def test_captured_paged_steps_keep_their_memory(torch, lib, name):
    """Two captured steps, replayed on two streams at once after larger eager passes whose memory,
    and what it replaced, went to other tensors: the bits of the eager steps."""
    p = Paged(torch, name)
    states = [p.state(b) for b in (3, 4)]
    want = [p.chunk(s, 40, 40 + n)[0] for s, n in zip(states, (1, 4))]
    steps = [s.args for s in states]
    side, graphs, outs = torch.cuda.Stream(), [], []
    for a in steps:
        gr = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(gr, stream=side):
            outs.append(p.call(a)[0])
        graphs.append(gr)
    other = p.state(9)
    p.chunk(other, 40, 120)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    taken = [torch.full((n,), 0x5A, dtype=torch.uint8, device="cuda") for n in [1 << 20] * 40 + [1 << 24] * 10]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        p.chunk(other, 40, 100)  # and an eager pass beside them
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
    assert all(bool((t == 0x5A).all()) for t in taken)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward_paged_with_several_axes(torch, lib, quantized, interleaved):
    """Three axes at the same positions are one axis, bit for bit; at others they are not."""
    p = Paged(torch, "w8a16")
    out = []
    for axes in (1, 3):
        s = p.state(6, quantized)
        p.chunk(s, 40, 50)
        ids, pos, batch, caches = s.args
        if axes == 1:
            out.append(p.call(s.args)[0])
        else:
            kw = dict(sections=(24, 20, 20), interleaved=interleaved)
            out.append(p.call((ids, pos.expand(3, -1).contiguous(), batch, caches), **kw)[0])
            out.append(p.call((ids, torch.stack([pos, pos + 3, pos // 2]).contiguous(), batch, caches), **kw)[0])
    assert torch.equal(out[0], out[1]) and not torch.equal(out[0], out[2])


# ------------------------------------------------------------------ graphs over the shared workspaces
def fill(torch):
    """Free blocks of the allocator, taken and filled."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    return [torch.full((n,), 0x5A, dtype=torch.uint8, device="cuda") for n in [1 << 20] * 40 + [1 << 24] * 10]


@pytest.mark.parametrize("eager_first", [True, False])
def test_a_captured_decode_step_after_a_larger_prefill(torch, lib, eager_first):
    """The stage's workspace grows behind a captured step, or is first asked for by one."""
    from dial_cuda.model import Decoder, ModelConfig
    dec = Decoder(ModelConfig(**CONFIGS["w8a16"]), n_slots=2, max_seq=256)
    i32 = dict(dtype=torch.int32, device="cuda")
    ids, pos, slot, out = torch.tensor([7], **i32), torch.tensor([0], **i32), torch.tensor([1], **i32), torch.empty(1, **i32)
    hidden = torch.empty((1, dec.cfg.hidden), device="cuda", dtype=dec.stage.dt)
    if eager_first:
        dec.decode_step(ids, pos, slot, 1, out, hidden=hidden)
    gr = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(gr):
        dec.decode_step(ids, pos, slot, 1, out, hidden=hidden)
    prompt = torch.arange(200, **i32)
    first = dec.prefill(prompt, slot=0)
    assert torch.equal(dec.prefill(prompt, slot=0), first)
    taken = fill(torch)
    for _ in range(3):
        gr.replay()
        assert torch.equal(dec.prefill(prompt, slot=0), first)
    torch.cuda.synchronize()
    got, bits = out.clone(), hidden.clone()
    dec.decode_step(ids, pos, slot, 1, out, hidden=hidden)
    assert torch.equal(out, got) and torch.equal(hidden, bits)
    assert all(bool((t == 0x5A).all()) for t in taken)


def test_a_captured_linear_after_a_larger_call(torch, lib):
    g = gen(torch, 8)
    lin = lib.GgufLinear.quantize(torch.randn((512, 1152), generator=g, device="cuda") * 0.05, lib.Q4_0)
    x, big = (torch.randn((m, 1152), generator=g, device="cuda").half() for m in (9, 3000))
    side, gr = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    out = torch.empty((9, 512), device="cuda", dtype=torch.float16)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        want = lin.forward(x)
    torch.cuda.synchronize()
    with torch.cuda.graph(gr, stream=side):
        lin.forward(x, out)
    with torch.cuda.stream(side):
        lin.forward(big)
    taken = fill(torch)
    for _ in range(3):
        out.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert all(bool((t == 0x5A).all()) for t in taken)


def test_forward_paged_with_a_linear_wider_than_a_shared_workspace_serves(torch, lib):
    """gate_up of 262784 outputs: its counters are longer than the shared ones."""
    CONFIGS["wide"] = dict(n_layers=2, hidden=384, intermediate=131392, n_heads=1, n_kv_heads=1, vocab=100, qk_norm=False,
                           weight_format=8, head_format=8)
    try:
        p = Paged(torch, "wide")
    finally:
        del CONFIGS["wide"]
    s = p.state(7)
    first = p.chunk(s, 40, 42)[0]
    assert torch.isfinite(first).all()
    for _ in range(3):
        assert torch.equal(p.call(s.args)[0], first)
