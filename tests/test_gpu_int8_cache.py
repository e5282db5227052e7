"""int8 paged cache on the GPU: writes and decode attention against the definition in 64 bits."""
import pytest
import torch

import _int8 as R
from axonml_b200.ops import paged

pytestmark = pytest.mark.gpu


def _table(need, extra=2, seed=0):
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(sum(need) + extra, generator=g).tolist()
    table, at = torch.zeros(len(need), max(need + [1]), dtype=torch.int32), 0
    for b, c in enumerate(need):
        table[b, :c] = torch.tensor(perm[at:at + c], dtype=torch.int32)
        at += c
    return table, sum(need) + extra


@pytest.mark.parametrize("lens,starts", [([1], [0]), ([1] * 5, [0, 15, 16, 33, 7]), ([40, 0, 3, 17], [0, 5, 30, 31]), ([300, 1, 77], [9, 0, 64]),
                                         ([1] * 70, [i * 3 for i in range(70)])])
@pytest.mark.parametrize("Hkv,P,D", [(1, 16, 64), (3, 32, 128), (2, 64, 256), (8, 16, 128), (2, 16, 80)])
def test_write(lens, starts, Hkv, P, D, kernel_status):
    table, pages = _table([(s + n + P - 1) // P for s, n in zip(starts, lens)])
    T = sum(lens)
    k, v = torch.randn(T + 3, Hkv, D, device="cuda").bfloat16(), (torch.randn(T + 3, Hkv, D, device="cuda") * 3).bfloat16()
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    kc, vc, ka, va = R.make_cache(pages, Hkv, P, D, "cuda")
    want_k = R.write(kc.double(), ka.double(), k, table.tolist(), starts, cu.tolist())
    want_v = R.write(R.v_rows(vc).double(), va.double(), v, table.tolist(), starts, cu.tolist())
    st = torch.tensor(starts, dtype=torch.int32).cuda()
    for _ in range(2):                                    # rows behind the last sequence are ignored; again changes nothing
        paged.kv_write_int8(k, v, kc, vc, ka, va, table.cuda(), st, cu.cuda())
        assert torch.equal(ka.double(), want_k[1]) and torch.equal(kc.double(), want_k[0])
        assert torch.equal(va.double(), want_v[1]) and torch.equal(R.v_rows(vc).double(), want_v[0])


def test_write_without_offsets_strided_fp32_and_zeros(kernel_status):
    Hkv, P, D, B = 2, 16, 64, 4
    table, pages = _table([3] * B)
    qkv = torch.randn(B * 6, 2 * Hkv + 5, D, device="cuda")
    qkv[:6] = 0.0                                         # a sequence of zeros
    for dt in (torch.float32, torch.bfloat16):
        x = qkv.to(dt)
        k, v = x[:, 5:5 + Hkv], x[:, 5 + Hkv:]            # slices of a fused projection
        caches = R.make_cache(pages, Hkv, P, D, "cuda", seed=1)
        cpu = [t.cpu() for t in caches]
        st = torch.tensor([0, 3, 30, 14], dtype=torch.int32)
        paged.kv_write_int8(k, v, *caches, table.cuda(), st.cuda())
        paged.kv_write_int8(k.cpu(), v.cpu(), *cpu, table, st)
        for a, b in zip(caches, cpu):
            assert torch.equal(a.cpu(), b)


def test_write_reports_what_does_not_fit():
    """Bad rows are skipped and reported; the others are written."""
    from axonml_b200 import _native as N
    Hkv, P, D = 2, 16, 64
    k = torch.randn(3, Hkv, D, device="cuda").bfloat16()
    for bad_start, bad_page in ((-1, 0), (16, 0), (0, 99), (0, -1)):
        kc, vc, ka, va = R.make_cache(4, Hkv, P, D, "cuda")
        before = [t.clone() for t in (kc, vc, ka, va)]
        table = torch.tensor([[1], [bad_page], [2]], dtype=torch.int32, device="cuda")
        st = torch.tensor([0, bad_start, 0], dtype=torch.int32, device="cuda")
        paged.kv_write_int8(k, k, kc, vc, ka, va, table, st)
        with pytest.raises(N.KernelTimeout):
            N.check_status()
        for t, o in zip((kc, vc, ka, va), before):
            assert torch.equal(t[0], o[0]) and torch.equal(t[3], o[3])
        assert ka[1].eq(k[0].float().abs().amax(-1)).all() and ka[2].eq(k[2].float().abs().amax(-1)).all()


def _attend(B, Hkv, G, D, P, ctx, seed=0, spare=0):
    table, pages = _table([(n + P - 1) // P for n in ctx], seed=seed)
    if spare:
        table = torch.cat([table, torch.full((B, spare), -7, dtype=torch.int32)], 1)      # entries past a context are not read
    kc, vc, ka, va = R.make_cache(pages, Hkv, P, D, "cuda", seed=seed)
    q = torch.randn(B, Hkv * G, D, device="cuda").bfloat16()
    cl = torch.tensor(ctx, dtype=torch.int32).cuda()
    got = paged.decode_attention_int8(q, kc, vc, ka, va, table.cuda(), cl)
    want, off = R.attention(q, kc, R.v_rows(vc), ka, va, table.tolist(), ctx, R.default_scale(D))
    assert got.dtype == torch.bfloat16
    assert ((got.double() - want).abs() <= off + torch.finfo(torch.bfloat16).eps / 2 * (want.abs() + off)).all()
    return got


@pytest.mark.parametrize("Hkv,G,D,P", [(8, 4, 128, 16), (1, 1, 64, 16), (2, 8, 128, 32), (3, 5, 64, 64), (2, 16, 128, 16), (1, 37, 128, 16),
                                       (2, 2, 256, 16), (1, 12, 256, 32), (4, 7, 64, 16), (16, 1, 128, 16)])
@pytest.mark.parametrize("ctx", [[1], [16], [17], [777], [0], [0, 5, 0, 0, 300, 64, 0], [2000, 3, 1000]])
@pytest.mark.parametrize("spare", [2, 9000])             # short tables: a cluster a head; long ones: even shares and a merge
def test_attention(Hkv, G, D, P, ctx, spare, kernel_status):
    got = _attend(len(ctx), Hkv, G, D, P, ctx, spare=spare)
    for b, n in enumerate(ctx):
        if n == 0:
            assert got[b].eq(0).all()


def test_attention_many_sequences_and_a_long_one(kernel_status):
    g = torch.Generator().manual_seed(3)
    _attend(300, 2, 4, 128, 16, [int(x) for x in torch.randint(0, 90, (300,), generator=g)], seed=3)
    _attend(2, 1, 8, 64, 16, [60000, 11], seed=4)
    _attend(40, 8, 4, 128, 16, [int(x) for x in torch.randint(1, 2500, (40,), generator=g)], seed=5)


@pytest.mark.parametrize("long_table", [False, True])
def test_attention_extreme_scores_and_scales(long_table, kernel_status):
    """One token that takes all the weight, q rows of very different sizes, a zero q, pages of zero magnitude."""
    Hkv, G, D, P, n = 2, 4, 128, 16, 200
    table, pages = _table([(n + P - 1) // P])
    if long_table:
        table = torch.cat([table, torch.zeros(1, 9000, dtype=torch.int32)], 1)
    kc, vc, ka, va = R.make_cache(pages, Hkv, P, D, "cuda", seed=9)
    q = torch.randn(1, Hkv * G, D, device="cuda").bfloat16()
    q[0, 0] *= 1e4
    q[0, 1] *= 1e-6
    q[0, 2] = 0
    q[0, 3, ::2] *= 1e-5
    ka[table[0, 3]] = 0.0
    va[table[0, 4]] = 0.0
    va[table[0, 5]] *= 1000
    cl = torch.tensor([n], dtype=torch.int32).cuda()
    for scale in (None, 0.5, 1e-4, -0.3, 0.0):
        got = paged.decode_attention_int8(q, kc, vc, ka, va, table.cuda(), cl, scale)
        want, off = R.attention(q, kc, R.v_rows(vc), ka, va, table.tolist(), [n], R.default_scale(D) if scale is None else scale)
        assert ((got.double() - want).abs() <= off + torch.finfo(torch.bfloat16).eps / 2 * (want.abs() + off)).all()
    # a page that is not finite reaches its own sequence and head only
    ka[table[0, 0], 1] = float("nan")
    got = paged.decode_attention_int8(q, kc, vc, ka, va, table.cuda(), cl)
    assert got[0, :G].isfinite().all() and got[0, G:].isnan().any()
    # and not where it lies behind the context
    cl16 = torch.tensor([16], dtype=torch.int32).cuda()
    ka[table[0, 0], 1] = 1.0
    va[table[0, 1]] = float("inf")
    assert paged.decode_attention_int8(q, kc, vc, ka, va, table.cuda(), cl16).isfinite().all()


@pytest.mark.parametrize("width", [0, 9000])
def test_attention_reports_bad_pages_and_contexts(width):
    from axonml_b200 import _native as N
    kc, vc, ka, va = R.make_cache(4, 2, 16, 64, "cuda")
    q = torch.randn(3, 4, 64, device="cuda").bfloat16()
    cl = torch.tensor([20, 30, 9], dtype=torch.int32).cuda()
    for table, ctx in (([[0, 1], [2, 99], [3, 0]], cl), ([[0, 1], [-1, 2], [3, 0]], cl), ([[0, 1], [2, 1], [3, 0]], cl + torch.tensor([0, 90 + 16 * width, 0]).cuda().int())):
        t = torch.cat([torch.tensor(table, dtype=torch.int32), torch.zeros(3, width, dtype=torch.int32)], 1)
        got = paged.decode_attention_int8(q, kc, vc, ka, va, t.cuda(), ctx)
        with pytest.raises(N.KernelTimeout):
            N.check_status()
        for b in (0, 2):
            want, off = R.attention(q[b:b + 1], kc, R.v_rows(vc), ka, va, table[b:b + 1], [int(cl[b])], R.default_scale(64))
            assert ((got[b:b + 1].double() - want).abs() <= off + 2.0 ** -8 * (want.abs() + off)).all()


@pytest.mark.parametrize("D,dt,err", [(96, torch.bfloat16, ValueError), (64, torch.float32, TypeError)])
def test_attention_gpu_refusals(D, dt, err):
    c = R.make_cache(2, 1, 16, D, "cuda")
    with pytest.raises(err):
        paged.decode_attention_int8(torch.zeros(1, 1, D, device="cuda", dtype=dt), *c, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                                    torch.ones(1, dtype=torch.int32, device="cuda"))


def test_write_then_attend_in_a_graph_and_on_another_stream(kernel_status):
    """Decode steps captured once and replayed: the write feeds the attention; two graphs share one cache in turn."""
    Hkv, G, D, P, B = 2, 4, 128, 16, 3
    table, pages = _table([4] * B)
    caches, eager = R.make_cache(pages, Hkv, P, D, "cuda", zero=True), R.make_cache(pages, Hkv, P, D, "cuda", zero=True)
    tab = table.cuda()
    x = torch.zeros(2, B, Hkv, D, device="cuda").bfloat16()
    q = torch.zeros(B, Hkv * G, D, device="cuda").bfloat16()
    pos = torch.zeros(B, dtype=torch.int32, device="cuda")

    def step(c):
        paged.kv_write_int8(x[0], x[1], *c, tab, pos)
        return paged.decode_attention_int8(q, *c, tab, pos + 1)
    step([t.clone() for t in caches])
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(caches)
        graphs.append((g, out))
    for t in caches:
        t.zero_()
    side = torch.cuda.Stream()
    for n in range(40):
        x.copy_(torch.randn(2, B, Hkv, D))
        q.copy_(torch.randn(B, Hkv * G, D))
        pos.fill_(n)
        g, out = graphs[n % 2]
        g.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = step(eager)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, want)
    for a, b in zip(caches, eager):
        assert torch.equal(a, b)


def test_captured_branches_memsets_and_copies(kernel_status):
    """The operators as first and as joining nodes of a captured fork, behind a memset and a copy, replayed several times."""
    from axonml_b200.ops import int8 as I
    x = torch.randn(300, 512, device="cuda").bfloat16()
    w = torch.ones(512, device="cuda").bfloat16()
    W = I.Int8Weight.from_dense(torch.randn(384, 512, device="cuda"))
    src, buf = torch.zeros_like(x), torch.zeros_like(x)

    def steps(side):
        here = torch.cuda.current_stream()
        buf.zero_()
        a = I.rms_norm_int8(buf, w, residual=x)               # behind a memset
        side.wait_stream(here)
        with torch.cuda.stream(side):
            b = I.int8_linear(*I.quantize_int8(x), W.q, W.scale)          # first of a branch
        buf.copy_(src)
        c = I.int8_linear(a[0], a[1], W.q, W.scale)           # behind a copy, beside the branch
        here.wait_stream(side)
        d = I.rms_norm_int8(c, torch.ones(384, device="cuda").bfloat16(), residual=b)     # joins both
        return [*a, b, c, *d]
    side = torch.cuda.Stream()
    steps(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = steps(side)
    for _ in range(3):
        x.copy_(torch.randn(300, 512))
        src.copy_(torch.randn(300, 512))
        for _ in range(4):
            g.replay()
        torch.cuda.synchronize()
        want = steps(side)
        torch.cuda.synchronize()
        for p, q in zip(out, want):
            assert torch.equal(p, q)


@pytest.mark.parametrize("long", [0, 1])
def test_two_calls_at_once(long, kernel_status):
    """The same operators on two streams at the same time, each with its own inputs."""
    Hkv, G, D, P = 4, 4, 128, 16
    ctx = [1500, 3, 900]
    table, pages = _table([(n + P - 1) // P for n in ctx])
    table = torch.cat([table, torch.zeros(3, 5000 * long, dtype=torch.int32)], 1)
    cl, tab = torch.tensor(ctx, dtype=torch.int32).cuda(), table.cuda()
    sets = [R.make_cache(pages, Hkv, P, D, "cuda", seed=s) + [torch.randn(3, Hkv * G, D, device="cuda").bfloat16()] for s in (1, 2)]
    alone = [paged.decode_attention_int8(c[4], *c[:4], tab, cl) for c in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (c, s) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(s):
                got[i].append(paged.decode_attention_int8(c[4], *c[:4], tab, cl))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, alone[i]) for x in got[i])


def test_capture_before_the_first_call_is_refused():
    """The status word is made outside captures."""
    from axonml_b200 import _native as N
    saved, words = dict(N._STATUS_PTR), dict(N._STATUS)
    W = torch.zeros(32, 32, dtype=torch.int8, device="cuda")
    s = torch.ones(32, device="cuda")
    from axonml_b200.ops import int8 as I
    g = torch.cuda.CUDAGraph()
    try:
        N._STATUS_PTR.clear()
        N._STATUS.clear()
        with pytest.raises(N.NativeError):
            with torch.cuda.graph(g):
                I.int8_linear(W, s, W, s)
    finally:
        N._STATUS_PTR.update(saved)
        N._STATUS.update(words)
    torch.cuda.synchronize()


def _gpu_model(**kw):
    from axonml_b200.llm import LLaMAConfig
    from axonml_b200.quant import QuantType
    from axonml_b200.server import QuantizedLlama
    cfg = LLaMAConfig(vocab_size=20000, hidden_size=1024, intermediate_size=2048, num_hidden_layers=2, num_attention_heads=8,
                      num_key_value_heads=4, max_position_embeddings=256)
    return QuantizedLlama.from_random(cfg, None, device="cuda", std=0.05, proj_type=QuantType.Q4_K, **kw)


@pytest.mark.parametrize("weights,kv", [(True, torch.int8), (False, torch.int8), (True, torch.bfloat16)])
def test_engine_in_eight_bits(weights, kv, kernel_status, monkeypatch):
    """Every operator call of a prefill and a decode step against 64 bits; decoding with graphs against the same without."""
    from axonml_b200.server import LLMEngine, PagedKVCache
    model8 = _gpu_model()
    prompts = [[(11 * i + j) % 19000 for j in range(20)] for i in range(5)]
    cache = PagedKVCache(2, 16, 16, model8.hkv, model8.hd, 5, 3, model8.device, dtype=kv)
    if weights:
        model8.to_int8()
    slots = [cache.allocate_seq() for _ in prompts]
    for s in slots:
        cache.reserve(s, 21)
    with monkeypatch.context() as mp, torch.no_grad():
        rec = R.Recorder(mp)
        model8.prefill(torch.tensor(prompts, device="cuda"), cache, slots)
        model8.decode(torch.arange(5, device="cuda"), cache, torch.tensor(slots, dtype=torch.int32, device="cuda"),
                      torch.full((5,), 20, dtype=torch.int32, device="cuda"))
    assert len(rec.calls) == 2 * 2 * ((8 if weights else 0) + (1 if kv == torch.int8 else 0)) + (2 if kv == torch.int8 else 0)
    rec.check()
    monkeypatch.setenv("AXONML_DECODE_GRAPHS", "1")
    a = LLMEngine(model8, max_batch=5, max_context=64, page_size=16, kv_dtype=kv).generate(prompts, 24)
    monkeypatch.setenv("AXONML_DECODE_GRAPHS", "0")
    b = LLMEngine(model8, max_batch=5, max_context=64, page_size=16, kv_dtype=kv).generate(prompts, 24)
    assert all(len(x) == 24 for x in a + b)
    if weights:                                           # the Q4_K product adds split sums in no fixed order, the int8 one is exact
        assert a == b


@pytest.mark.parametrize("n,ctx", [(1, [1]), (40, [40, 17]), (700, [700, 16, 333])])
@pytest.mark.parametrize("spare", [0, 9000])
def test_attention_of_scores_far_below_zero(n, ctx, spare, kernel_status):
    c, q, table, want = R.far_below(n, ctx, "cuda")
    table = torch.cat([table, torch.zeros(len(ctx), spare, dtype=torch.int32, device="cuda")], 1)
    got = paged.decode_attention_int8(q, *c, table, torch.tensor(ctx, dtype=torch.int32).cuda())
    assert ((got.double() - want).abs() <= R.far_below_off(want, q.dtype)).all()


def test_write_at_the_largest_positions(kernel_status):
    """The last page ends at position 2^31: all but its last slot can be written."""
    P, width = 1 << 20, 2048
    table = torch.zeros(1, width, dtype=torch.int32)
    k, v = torch.randn(16, 1, 16).bfloat16(), torch.randn(16, 1, 16).bfloat16()
    cpu = R.make_cache(1, 1, P, 16, "cpu", seed=2)
    gpu = [t.cuda() for t in cpu]
    st = torch.tensor([2 ** 31 - 17], dtype=torch.int32)
    paged.kv_write_int8(k, v, *cpu, table, st)
    paged.kv_write_int8(k.cuda(), v.cuda(), *gpu, table.cuda(), st.cuda())
    for a, b in zip(gpu, cpu):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("B", [1, 33, 2000])
def test_write_of_one_token_each_with_bad_rows(B):
    """Without offsets a token's page is its row's: a bad row leaves the others alone."""
    from axonml_b200 import _native as N
    Hkv, P, D = 2, 16, 64
    k, v = torch.randn(B, Hkv, D, device="cuda").bfloat16(), torch.randn(B, Hkv, D, device="cuda").bfloat16()
    gpu = R.make_cache(B, Hkv, P, D, "cuda", seed=4)
    st = torch.arange(B, dtype=torch.int32) % 16
    st[0] = -1
    want = [t.cpu() for t in gpu]
    table = torch.arange(B, dtype=torch.int32)[:, None]
    paged.kv_write_int8(k, v, *gpu, table.cuda(), st.cuda())
    with pytest.raises(N.KernelTimeout):
        N.check_status()
    if B > 1:
        paged.kv_write_int8(k[1:].cpu(), v[1:].cpu(), *want, table[1:], st[1:])
    for a, b in zip(gpu, want):
        assert torch.equal(a.cpu(), b)


def test_too_many_tokens_are_refused():
    c = R.make_cache(1, 1, 16, 64, "cuda")
    k = torch.zeros(1, 1, 64, device="cuda").bfloat16().expand((1 << 30) + 1, 1, 64)
    with pytest.raises(ValueError):
        paged.kv_write_int8(k, k, *c, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"))


def test_attention_from_several_threads(kernel_status):
    """Batches of very different size from host threads at the same time."""
    import threading
    cases = []
    for i, B in enumerate((1, 3000, 40, 8000)):
        c = R.make_cache(B, 1, 16, 64, "cuda", seed=i)
        q = torch.randn(B, 1, 64, device="cuda").bfloat16()
        table = torch.cat([torch.arange(B, dtype=torch.int32)[:, None], torch.zeros(B, 600, dtype=torch.int32)], 1).cuda()
        cl = (torch.arange(B, dtype=torch.int32) % 17).cuda()
        cases.append((q, *c, table, cl))
    torch.cuda.synchronize()
    got, errors = [[] for _ in cases], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i].append(paged.decode_attention_int8(*cases[i]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, x in zip(cases, got):
        alone = paged.decode_attention_int8(*a)
        assert len(x) == 10 and all(torch.equal(y, alone) for y in x)


@pytest.mark.parametrize("B,spare", [(1024, 0), (1025, 700), (2500, 0), (2500, 700)])
def test_attention_of_very_many_sequences(B, spare, kernel_status):
    g = torch.Generator().manual_seed(B)
    _attend(B, 1, 4, 64, 16, [int(x) for x in torch.randint(0, 60, (B,), generator=g)], seed=6, spare=spare)


@pytest.mark.parametrize("B", [129, 2000])
def test_write_of_very_many_sequences(B, kernel_status):
    """Rows of zero, one and more tokens, found by a search over the offsets."""
    Hkv, P, D = 1, 16, 64
    g = torch.Generator().manual_seed(B)
    lens = [int(x) for x in torch.tensor([0, 0, 1, 1, 2, 40])[torch.randint(0, 6, (B,), generator=g)]]
    starts = [int(x) for x in torch.randint(0, 33, (B,), generator=g)]
    table, pages = _table([(s + n + P - 1) // P for s, n in zip(starts, lens)])
    first = 3                                              # rows before the first sequence are ignored too
    T = first + sum(lens) + 2
    k, v = torch.randn(T, Hkv, D).bfloat16(), torch.randn(T, Hkv, D).bfloat16()
    cu = first + torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    cpu = R.make_cache(pages, Hkv, P, D, "cpu")
    gpu = [t.cuda() for t in cpu]
    st = torch.tensor(starts, dtype=torch.int32)
    paged.kv_write_int8(k, v, *cpu, table, st, cu.int())
    paged.kv_write_int8(k.cuda(), v.cuda(), *gpu, table.cuda(), st.cuda(), cu.int().cuda())
    for a, b in zip(gpu, cpu):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("lens,starts", [([1], [100]), ([100, 0, 7], [47, 5, 48]), ([3] * 40, [i * 5 for i in range(40)])])
@pytest.mark.parametrize("cu", [True, False])
def test_pages_of_no_power_of_two(lens, starts, cu, kernel_status):
    if not cu and len(set(lens)) > 1:
        lens = [5] * len(lens)
    Hkv, P, D = 2, 48, 64
    table, pages = _table([(s + n + P - 1) // P for s, n in zip(starts, lens)])
    k, v = torch.randn(sum(lens), Hkv, D).bfloat16(), torch.randn(sum(lens), Hkv, D).bfloat16()
    off = torch.tensor([0] + lens).cumsum(0).int() if cu else None
    cpu = R.make_cache(pages, Hkv, P, D, "cpu")
    gpu = [t.cuda() for t in cpu]
    st = torch.tensor(starts, dtype=torch.int32)
    paged.kv_write_int8(k, v, *cpu, table, st, off)
    paged.kv_write_int8(k.cuda(), v.cuda(), *gpu, table.cuda(), st.cuda(), off.cuda() if cu else None)
    for a, b in zip(gpu, cpu):
        assert torch.equal(a.cpu(), b)
    _attend(len(lens), Hkv, 4, D, P, [s + n for s, n in zip(starts, lens)], seed=7)


@pytest.mark.parametrize("spare", [0, 9000])
def test_cache_of_more_than_2_to_the_31_bytes(spare, kernel_status):
    """Pages at both ends of caches of 2.4 GB each, against the same pages in a small cache."""
    Hkv, G, P, D, pages = 8, 4, 16, 128, 150_000
    kc = torch.empty(pages, Hkv, P, D, dtype=torch.int8, device="cuda")
    vc = torch.empty(pages, Hkv, 1, D, 16, dtype=torch.int8, device="cuda")
    ka, va = torch.zeros(pages, Hkv, device="cuda"), torch.zeros(pages, Hkv, device="cuda")
    far = [pages - 1, 0, pages - 2, 131072, 131071, 1, 140_000, 149_000]
    k, v = torch.randn(2 * 60, Hkv, D, device="cuda").bfloat16(), torch.randn(2 * 60, Hkv, D, device="cuda").bfloat16()
    q = torch.randn(2, Hkv * G, D, device="cuda").bfloat16()
    st, cl = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.full((2,), 60, dtype=torch.int32, device="cuda")
    got = []
    for caches, ids in (((kc, vc, ka, va), far), (R.make_cache(8, Hkv, P, D, "cuda"), list(range(8)))):
        table = torch.zeros(2, 4 + spare, dtype=torch.int32)
        table[:, :4] = torch.tensor(ids).view(2, 4)
        paged.kv_write_int8(k, v, *caches, table.cuda(), st)
        got.append((paged.decode_attention_int8(q, *caches, table.cuda(), cl), caches, ids))
    (a, big, ids), (b, small, _) = got
    assert torch.equal(a, b)
    for x, y in zip(big, small):
        assert torch.equal(x[ids][[0, 1, 2, 4, 5, 6]], y[[0, 1, 2, 4, 5, 6]])
    assert big[2].count_nonzero() == 8 * Hkv                        # and no other page's magnitude


def test_gradients_and_copies_of_unaligned_rows(kernel_status):
    """Rows off the 16-byte grid and reversed heads are copied; what requires a gradient is refused."""
    Hkv, P, D = 2, 16, 64
    c, ref = R.make_cache(2, Hkv, P, D, "cuda", zero=True), R.make_cache(2, Hkv, P, D, "cuda", zero=True)
    wide = torch.randn(5, Hkv, D + 3, device="cuda").bfloat16()
    table, st = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = wide[..., 3:], wide[..., 1:D + 1].flip(1).transpose(0, 1).contiguous().transpose(0, 1)
    paged.kv_write_int8(k, v, *c, table, st)
    paged.kv_write_int8(k.contiguous(), v.contiguous(), *ref, table, st)
    for a, b in zip(c, ref):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        paged.kv_write_int8(k.detach().requires_grad_(), v, *c, table, st)
    with pytest.raises(RuntimeError):
        paged.decode_attention_int8(torch.randn(1, 2, D, device="cuda").bfloat16().requires_grad_(), *c, table, st + 5)
