"""The language-model operators at the edges of what their documentation allows:
values, streams and tensors that the shapes of test_gpu_lm_ops.py do not bring.
"""
import pytest
import torch

from test_gpu_lm_ops import F8, Batch, close, codes, product_ref, product_tol, randn, vxb  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- rms norm --

@pytest.mark.parametrize("C", [4096, 1000, 77])
def test_rms_norm_codes_are_the_rounded_quotients(vxb, C):  # noqa: F811
    """scale = max|y| / 448 (by the rounded 1 / 448, as torch does it: bit for bit) and code = e4m3(y / scale) of
    the fp32 output y, where a quotient is off by two roundings of 2^-24 at most (blocks of size 2^-60 to 2^60, so that no
    quotient is special)."""
    kb = -(-C // 128)
    x = randn(1, 200, C)
    w = (randn(2, C) * 2.0 ** torch.linspace(-60, 60, kb, device="cuda").repeat_interleave(128)[:C]).contiguous()
    y = torch.empty_like(x)
    vxb.rms_norm(x, w, y)
    q, s = torch.empty(200, C, dtype=F8, device="cuda"), torch.empty(200, kb, device="cuda")
    vxb.rms_norm(x, w, q, y_scale=s)
    top = torch.nn.functional.pad(y, (0, kb * 128 - C)).view(200, kb, 128).abs().amax(2)
    assert torch.equal(s, top / 448)
    by = s.repeat_interleave(128, 1)[:, :C]
    quotient = y.double() / by.double()
    lo, hi = ((quotient * (1 + d)).float().to(F8).view(torch.uint8) for d in (-(2.0 ** -23), 2.0 ** -23))
    got = q.view(torch.uint8)
    assert ((got == lo) | (got == hi)).all()


def test_rms_norm_codes_of_the_largest_values(vxb):  # noqa: F811
    """Blocks whose maximum lies above 2^126 (8.5e37) keep their codes; a block with an infinity has the
    scale infinity, zeros for what is finite and NaN for what is not."""
    x = torch.ones(3, 512, device="cuda")
    x[:, 1::2] = -1
    w = torch.ones(512, device="cuda")
    w[:128], w[128:256], w[256] = 2e38, 8e37, float("inf")
    y, q, s = torch.empty_like(x), torch.empty(3, 512, dtype=F8, device="cuda"), torch.empty(3, 4, device="cuda")
    vxb.rms_norm(x, w, y)
    vxb.rms_norm(x, w, q, y_scale=s)
    for b in (0, 1, 3):
        assert torch.equal(q[:, 128 * b: 128 * b + 128].float(), 448 * x[:, :128])
        assert torch.equal(s[:, b], y[:, 128 * b] / 448)
    assert torch.isinf(s[:, 2]).all() and torch.isnan(q[:, 256].float()).all() and not q[:, 257:384].float().any()


# ------------------------------------------------------------- fp8 product --

@pytest.mark.parametrize("N", [1, 2, 16, 600])
def test_norm_and_product_in_turn_in_a_graph(vxb, N):  # noqa: F811
    """Products right behind the norms that write their operands, with nothing between them but the programmatic
    launch: new inputs at every replay, bit for bit what calls with a synchronisation between them give."""
    C, M, layers = 1024, 1024, 6
    ws = [codes(20 + 10 * i, M, C, 128) for i in range(layers)]
    gain = [randn(7 + i, C) + 1 for i in range(layers)]
    x = torch.empty(N, C, device="cuda")
    q, s = torch.empty(N, C, dtype=F8, device="cuda"), torch.empty(N, C // 128, device="cuda")
    y = torch.empty(N, M, device="cuda")

    def run(wait):
        src = x
        for (w, w_s), g in zip(ws, gain):  # one set of buffers: each pair overwrites what the last one read
            vxb.rms_norm(src, g, q, y_scale=s)
            wait()
            vxb.fp8_product(q, s, w, w_s, y)
            wait()
            src = y

    run(lambda: None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(lambda: None)
    for step in range(8):
        x.copy_(randn(100 + step, N, C, scale=1.0 + step))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        run(torch.cuda.synchronize)
        assert torch.equal(got, y)


PRODUCTS = [  # each way the product is formed: no tensor cores, weights as rows, tokens as rows, K split or not
    (1, 1024, 4096), (2, 2048, 129), (1, 8192, 8192), (3, 528, 70), (16, 1536, 1000), (31, 4096, 512), (64, 8192, 384),
    (77, 1536, 1001), (256, 1024, 64), (200, 4096, 1024), (129, 256, 130), (700, 512, 7000), (2500, 384, 2056)]


@pytest.mark.parametrize("N,K,M", PRODUCTS)
def test_fp8_product_error_as_a_whole(vxb, N, K, M):  # noqa: F811
    """The worst case of a long sum hides errors that matter; taken together, errors are as small as fp32's.
    A product of a block loses at most 2^-24 of the largest value in each of its 128 additions, and each of the
    blocks' additions 2^-24 of the sum."""
    x, xs = codes(1, N, K, 1)
    w, ws = codes(5, M, K, 128)
    y = torch.empty(N, M, device="cuda")
    vxb.fp8_product(x, xs, w, ws, y)
    ref, _ = product_ref(x, xs, w, ws, None)
    off = (y.double() - ref).square().mean().sqrt() / ref.square().mean().sqrt()
    assert float(off) <= (128 + 2 * -(-K // 128)) * 2.0 ** -24


@pytest.mark.parametrize("N,K,M", PRODUCTS)
def test_fp8_product_of_small_integers_is_exact(vxb, N, K, M):  # noqa: F811
    """Codes -2 .. 2 and scales 1/2, 1, 2: every sum is a multiple of 1/4 below 2^17 (64 blocks of 512 times 4), which
    fp32 holds, so nothing is rounded."""
    g = torch.Generator(device="cuda").manual_seed(N + K + M)

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda").float()

    x, w = ints(-2, 3, N, K).to(F8), ints(-2, 3, M, K).to(F8)
    xs, ws = 2.0 ** ints(-1, 2, N, -(-K // 128)), 2.0 ** ints(-1, 2, -(-M // 128), -(-K // 128))
    bias = ints(-8, 9, M)
    y = torch.empty(N, M, device="cuda")
    vxb.fp8_product(x, xs, w, ws, y, bias=bias)
    ref, _ = product_ref(x, xs, w, ws, bias)
    assert torch.equal(y.double(), ref)


# ------------------------------------------------------------ failed waits --

def test_expired_wait_is_reported_once_and_operators_go_on(vxb):  # noqa: F811
    x, xs = codes(1, 9, 1024, 1)
    w, ws = codes(5, 640, 1024, 128)
    a, y = (torch.empty(9, 640, device="cuda") for _ in range(2))
    vxb.fp8_product(x, xs, w, ws, a)
    vxb.operators_sync()
    side = torch.cuda.Stream()
    vxb.operators_wait_probe(1000, stream=side)
    vxb.fp8_product(x, xs, w, ws, y, stream=side)
    with pytest.raises(vxb.VxbError) as e:
        vxb.operators_sync(5000, stream=side)
    assert e.value.code == vxb.ERR_DEVICE_STATUS and "wait" in str(e.value)
    vxb.operators_sync(stream=side)  # read and cleared
    vxb.operators_sync()
    assert torch.equal(a, y)


def test_operators_sync_leaves_a_capture_alone(vxb):  # noqa: F811
    x, w = randn(1, 4, 256), torch.ones(256, device="cuda")
    a, y = torch.empty_like(x), torch.empty_like(x)
    vxb.rms_norm(x, w, a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        vxb.rms_norm(x, w, y)
        with pytest.raises(vxb.VxbError) as e:
            vxb.operators_sync()
    assert e.value.code == vxb.ERR_INVALID_ARGUMENT
    graph.replay()
    vxb.operators_sync()
    assert torch.equal(a, y)


def test_operators_sync_gives_up_at_its_timeout(vxb):  # noqa: F811
    vxb.operators_wait_probe(300000)
    with pytest.raises(vxb.VxbError) as e:
        vxb.operators_sync(10)
    assert e.value.code == vxb.ERR_TIMEOUT
    with pytest.raises(vxb.VxbError) as e:
        vxb.operators_sync()
    assert e.value.code == vxb.ERR_DEVICE_STATUS
    vxb.operators_sync()


# --------------------------------------------------------- paged attention --

@pytest.mark.parametrize("q_len", [1, 20])
def test_attention_non_finite_value_of_no_weight_in_a_part_of_its_own(vxb, q_len):  # noqa: F811
    """A value that a token sees reaches it whatever its weight, also where the keys are split and the part
    that holds it is outweighed by more than fp32's range."""
    b = Batch([q_len], [5000], 16, 2, 128, 64, torch.bfloat16)
    b.q.fill_(1.0)
    for j in range(5000 // 64 + 1):
        b.k[int(b.table[0, j])] = -30.0 if j < 16 else 0.0  # scores of -339 at the first 1024 keys, 0 elsewhere
    b.v[int(b.table[0, 1]), 3, 1, 7] = float("inf")
    assert vxb.lib().vxb_paged_attention_workspace(q_len, 1, 16, 2, 128, b.table.shape[1], 64) > 0
    out = b.run(vxb)
    bad = torch.zeros(q_len, 16, 128, dtype=torch.bool, device="cuda")
    bad[:, 8:, 7] = True
    assert torch.equal(~torch.isfinite(out), bad)


@pytest.mark.parametrize("q_len,Hq,Hk,D", [([600] + [1] * 20, 16, 2, 64), ([1] * 9 + [300] + [1] * 9, 8, 8, 128),
                                           ([60] + [1] * 40, 16, 2, 64), ([1] * 30 + [90, 0, 1], 4, 4, 128)])
@pytest.mark.parametrize("window", [0, 70])
def test_attention_of_chunks_and_single_tokens_in_one_call(vxb, q_len, Hq, Hk, D, window):  # noqa: F811
    """One kernel is chosen for the whole batch, from the average: right for both kinds of sequence on either side
    of the choice."""
    g = torch.Generator().manual_seed(len(q_len))
    kv = [n + int(torch.randint(0, 900, (), generator=g)) for n in q_len]
    b = Batch(q_len, kv, Hq, Hk, D, 16, torch.bfloat16, window=window, tail=2)
    b.run(vxb)
    b.check()


@pytest.mark.parametrize("q_len", [1, 3, 100])
def test_attention_of_broadcast_queries_and_caches(vxb, q_len):  # noqa: F811
    """Inputs may have strides of 0: one query for all tokens or heads, one key head or page for all."""
    def changes(b):
        yield {"q": b.q[:1].expand(q_len, 4, 64)}
        yield {"q": b.q[:, :1].expand(q_len, 4, 64)}
        yield {n: getattr(b, n)[:, :, :1].expand(-1, -1, 2, -1) for n in ("k", "v")}
        yield {n: randn(i, 1, 16, 2, 64, dtype=torch.bfloat16).expand(b.k.shape[0], 16, 2, 64)
               for i, n in enumerate(("k", "v"))}

    for i in range(4):
        b, ref = (Batch([q_len], [q_len + 60], 4, 2, 64, 16, torch.bfloat16) for _ in range(2))
        for n, t in list(changes(b))[i].items():
            setattr(b, n, t)
            setattr(ref, n, t.contiguous())
        assert torch.equal(b.run(vxb), ref.run(vxb))


def test_attention_output_quantised_by_the_caller_for_the_next_product(vxb):  # noqa: F811
    """The step between attention and output projection that no operator makes, in torch as a caller writes it."""
    b = Batch([5, 1, 70], [40, 33, 200], 4, 2, 64, 16, torch.bfloat16)
    o = b.run(vxb)
    blocks = o.view(76, -1, 128).float()
    o_scale = blocks.abs().amax(-1).clamp_(min=1e-30) / 448
    o8 = (blocks / o_scale[..., None]).view(76, -1).to(torch.float8_e4m3fn)
    w, ws = codes(5, 200, 256, 128)
    x = torch.empty(76, 200, device="cuda")
    vxb.fp8_product(o8, o_scale, w, ws, x)
    ref, mag = product_ref(o8, o_scale, w, ws, None)
    close(x, ref, product_tol(ref, mag, 256, torch.float32))
    whole, mag = (o.double().view(76, 256).abs() if i else o.double().view(76, 256) for i in (0, 1))
    wd = w.float().double() * ws.double().repeat_interleave(128, 0)[:200].repeat_interleave(128, 1)
    # a code is off by half a step of the value (2^-4) or of the smallest step (2^-10 scales)
    least = o_scale.double().repeat_interleave(128, 1) * 2.0 ** -10
    off = (torch.maximum(mag * 2.0 ** -4, least) * (1 + 2.0 ** -10)) @ wd.abs().t()
    assert ((x.double() - whole @ wd.t()).abs() <= off).all()


def test_outputs_of_any_nesting_and_refused_overlaps(vxb):  # noqa: F811
    b = Batch([3, 2], [40, 20], 4, 2, 64, 16, torch.bfloat16)
    ref = b.run(vxb).clone()
    b.out = torch.full((4, 5, 64), 5.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)  # heads outside
    assert torch.equal(b.run(vxb), ref)
    inv, pos = torch.from_numpy(vxb.rotary_frequencies(64)[0]).cuda(), torch.arange(5, device="cuda")
    plain = torch.empty_like(b.q)
    vxb.rotary(b.q, pos, inv, plain)
    outside = torch.empty(4, 5, 64, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    vxb.rotary(b.q, pos, inv, outside)
    assert torch.equal(plain, outside)
    for wrong in (torch.empty_like(ref[:1]).expand(5, 4, 64), torch.empty_like(ref[:, :1]).expand(5, 4, 64),
                  torch.empty(5 * 256, dtype=torch.bfloat16, device="cuda").as_strided((5, 4, 64), (128, 64, 1))):
        for call in (lambda: vxb.rotary(b.q, pos, inv, wrong),
                     lambda: vxb.paged_attention(b.q, b.k, b.v, b.table, b.cu, b.kv, wrong)):
            with pytest.raises(vxb.VxbError) as e:
                call()
            assert e.value.code == vxb.ERR_INVALID_ARGUMENT


# -------------------------------------------------------------- tensors --

def operator_calls(vxb):  # noqa: F811
    """(call, its tensors by name, those it writes) of every operator."""
    bf = torch.bfloat16
    x, w = randn(1, 4, 256, dtype=bf), randn(2, 256, dtype=bf)
    x8, xs = codes(3, 4, 256, 1)
    w8, ws = codes(4, 64, 256, 128)
    b = Batch([4], [40], 4, 2, 64, 16, bf)
    pos, slots = torch.arange(4, device="cuda"), torch.arange(4, device="cuda")
    inv = torch.from_numpy(vxb.rotary_frequencies(64)[0]).cuda()
    k = randn(5, 4, 2, 64, dtype=bf)
    e = torch.empty_like
    return [
        (vxb.rms_norm, dict(x=x, weight=w, y=e(x), residual=x.clone(), sum_out=e(x)), ("y", "sum_out")),
        (vxb.rms_norm, dict(x=x, weight=w, y=torch.empty(4, 256, dtype=F8, device="cuda"),
                            y_scale=torch.empty(4, 2, device="cuda")), ("y", "y_scale")),
        (vxb.fp8_product, dict(x=x8, x_scale=xs, w=w8, w_scale=ws, y=torch.empty(4, 64, device="cuda"),
                               bias=torch.zeros(64, device="cuda")), ("y",)),
        (vxb.rotary, dict(q=b.q, positions=pos, inv_freq=inv, q_out=e(b.q), k=k, k_out=e(k)), ("q_out", "k_out")),
        (vxb.rotary_append, dict(q=b.q, k=k, v=k.clone(), positions=pos, slots=slots, inv_freq=inv, q_out=e(b.q),
                                 k_cache=b.k, v_cache=b.v), ("q_out", "k_cache", "v_cache")),
        (vxb.paged_attention, dict(q=b.q, k_cache=b.k, v_cache=b.v, block_table=b.table, cu_q=b.cu, kv_len=b.kv,
                                   out=b.out), ("out",)),
    ]


def test_calls_raise_the_version_of_what_they_write(vxb):  # noqa: F811
    """autograd refuses a saved tensor that a call has overwritten since."""
    for call, t, written in operator_calls(vxb):
        before = {n: v._version for n, v in t.items()}
        call(**t)
        for n, v in t.items():
            assert (v._version > before[n]) == (n in written), (call.__name__, n)


def test_calls_refuse_to_lose_a_gradient(vxb):  # noqa: F811
    """No operator has a backward pass: with gradients on, a tensor that asks for one is refused."""
    for call, t, _ in operator_calls(vxb):
        for n, v in t.items():
            if not v.is_floating_point() or v.dtype == F8:
                continue
            with_grad = {**t, n: v.detach().requires_grad_()}
            with pytest.raises(vxb.VxbError) as e:
                call(**with_grad)
            assert e.value.code == vxb.ERR_INVALID_ARGUMENT and "gradient" in str(e.value)
            with torch.no_grad():
                call(**with_grad)
    with torch.inference_mode():  # (its tensors have no versions)
        for call, t, _ in operator_calls(vxb):
            call(**t)
    torch.cuda.synchronize()
