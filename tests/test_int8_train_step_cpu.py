"""LinearReluTrainStep's host logic with an int8 checkpoint of X, on CPU: its halves apart, what it keeps
between them, where its events lie, and the sum over two gloo ranks. The kernels are stood in for by plain
torch on CPU tensors, streams and events by recorders."""
import datetime
import socket
import types

import pytest
import torch

M, N, K = 24, 16, 40
BF16 = torch.bfloat16


class _Stream:
    def __init__(self, *a, **k):
        pass

    def wait_event(self, e):
        pass


class _Event:
    log: list = []

    def __init__(self, enable_timing=False):
        self.timing = enable_timing

    def record(self, stream=None):
        if self.timing:
            _Event.log.append("event")


def _plain(monkeypatch_setattr):
    """Plain CPU forms in the kernels' place; what runs is noted in the events' log."""
    from c3_b200 import linear, quant
    set_ = monkeypatch_setattr
    set_(torch.cuda, "Stream", _Stream)
    set_(torch.cuda, "Event", _Event)
    set_(torch.cuda, "current_stream", lambda *a: _Stream())
    set_(torch.cuda, "get_device_properties", lambda *a: types.SimpleNamespace(multi_processor_count=148))

    def forward(X, W, b, layout, Y, mask):
        _Event.log.append("forward")
        z = X.float() @ W.float().t() + b
        Y.copy_(z.clamp_min(0))
        bits = (z > 0).to(torch.int64)
        mask.copy_((bits << torch.arange(N)).sum(1, keepdim=True).to(torch.int32))

    def relu_mask_db(dY, mask, dZ, db):
        _Event.log.append("relu_mask_db")
        bits = (mask.to(torch.int64) >> torch.arange(N)) & 1
        dZ.copy_(dY * bits)
        db.copy_(dZ.float().sum(0))

    def quantize_rows(X, q, scale):
        _Event.log.append("quantize")
        big = X.float().abs().amax(1)
        scale.copy_(big / 127)
        q.copy_(torch.round(X.float() * 127 / big[:, None]))

    def grad_weight_int8(dZ, Xq, scale, dW):
        _Event.log.append("dw int8")
        dW.copy_(dZ.float().t() @ (Xq.float() * scale[:, None]))

    def grad_input(dZ, W, layout, dX):
        _Event.log.append("dx")
        dX.copy_(dZ.float() @ W.float())

    def gemm(dZ, X, a, b, epi, dW, M, N, K):
        _Event.log.append("dw bf16")
        dW.copy_(dZ.float().t() @ X.float())

    for name, fn in (("forward", forward), ("relu_mask_db", relu_mask_db), ("grad_weight_int8", grad_weight_int8),
                     ("grad_input", grad_input), ("gemm", gemm)):
        set_(linear, name, fn)
    set_(quant, "quantize_rows", quantize_rows)


def _inputs(seed):
    g = torch.Generator().manual_seed(seed)
    X = torch.randn((M, K), generator=g).to(BF16)
    dY = (torch.randn((M, N), generator=g) * 1e-2).to(BF16)
    g = torch.Generator().manual_seed(99)  # the same on every rank
    return X, (torch.randn((N, K), generator=g) * 0.1).to(BF16), torch.randn(N, generator=g), dY


@pytest.fixture
def plain(monkeypatch):
    _plain(monkeypatch.setattr)
    _Event.log = []


def test_the_halves_make_the_step_and_x_may_go(plain):
    from c3_b200.data_parallel import LinearReluTrainStep
    X, W, b, dY = _inputs(1)
    whole = LinearReluTrainStep(M, N, K, torch.device("cpu"), x_checkpoint="int8")
    whole(X, W, b, dY)
    halves = LinearReluTrainStep(M, N, K, torch.device("cpu"), x_checkpoint="int8")
    x = X.clone()
    assert halves.forward(x, W, b) is halves.Y
    x.fill_(float("nan"))
    assert halves.backward(W, dY) is halves.dX
    for name in ("Y", "mask", "dZ", "dX", "dW", "db", "Xq", "x_scale"):
        assert torch.equal(getattr(whole, name), getattr(halves, name)), name


def test_without_a_checkpoint_backward_needs_x(plain):
    from c3_b200.data_parallel import LinearReluTrainStep
    X, W, b, dY = _inputs(1)
    step = LinearReluTrainStep(M, N, K, torch.device("cpu"))
    step.forward(X, W, b)
    with pytest.raises(ValueError, match="needs the forward's X"):
        step.backward(W, dY)
    step.backward(W, dY, X)
    assert torch.equal(step.dW, (step.dZ.float().t() @ X.float()).to(BF16))


def test_the_recorded_phases_hold_all_of_the_step(plain):
    from c3_b200.data_parallel import LinearReluTrainStep
    X, W, b, dY = _inputs(1)
    step = LinearReluTrainStep(M, N, K, torch.device("cpu"), x_checkpoint="int8")
    events = step(X, W, b, dY, record=True)
    assert set(events.phases) == set(step.PHASES)
    assert _Event.log == ["event", "forward", "quantize", "event", "event", "relu_mask_db", "event", "event", "dw int8",
                          "event", "event", "dx", "event"]


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _rank(rank, world, port, queue):
    try:
        import torch.distributed as dist
        from c3_b200.data_parallel import LinearReluTrainStep
        _plain(setattr)
        dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world,
                                timeout=datetime.timedelta(seconds=60))
        X, W, b, dY = _inputs(rank)
        out = {}
        for chunks in (1, 2):
            step = LinearReluTrainStep(M, N, K, torch.device("cpu"), collective="group", chunks=chunks,
                                       x_checkpoint="int8", reserve_sms=20)
            step.forward(X, W, b)
            step.backward(W, dY)
            out[chunks] = (step.dW.float().numpy(), step.db.numpy().copy())
        queue.put((rank, out))
        dist.barrier()
        dist.destroy_process_group()
    except Exception as e:  # the parent sees it and does not wait
        queue.put((rank, repr(e)))


def test_two_ranks(plain):
    """Each rank's dW comes from its own checkpoint, and both end with the sum."""
    import torch.multiprocessing as mp
    from c3_b200.data_parallel import LinearReluTrainStep
    ctx = mp.get_context("spawn")
    queue, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=_rank, args=(r, 2, port, queue)) for r in range(2)]
    for p in procs:
        p.start()
    try:
        got = dict(queue.get(timeout=180) for _ in procs)
    finally:
        for p in procs:
            p.join(timeout=60)
            if p.is_alive():
                p.kill()
    dW, db = torch.zeros(N, K), torch.zeros(N)
    for r in range(2):
        X, W, b, dY = _inputs(r)
        step = LinearReluTrainStep(M, N, K, torch.device("cpu"), x_checkpoint="int8")
        step(X, W, b, dY)
        dW += step.dW.float()
        db += step.db
    for r in range(2):
        assert isinstance(got[r], dict), got[r]
        for chunks in (1, 2):
            w, v = (torch.from_numpy(t) for t in got[r][chunks])
            assert torch.equal(w, dW.to(BF16).float()) and torch.equal(v, db)  # two terms: one rounding each


@pytest.mark.gpu
@pytest.mark.parametrize("options", [{}, {"overlap_dx": True}, {"chunks": 2}])
def test_on_the_gpu(cuda_device, options):
    """The kernels in their place: X is overwritten as soon as `forward` has returned."""
    from c3_b200.data_parallel import LinearReluTrainStep
    m, n, k = 300, 256, 328
    g = torch.Generator(device=cuda_device).manual_seed(1)
    X, W, dY = (torch.randn(s, generator=g, device=cuda_device).to(BF16) for s in ((m, k), (n, k), (m, n)))
    b = torch.randn(n, generator=g, device=cuda_device)
    whole = LinearReluTrainStep(m, n, k, cuda_device, x_checkpoint="int8", **options)
    events = whole(X, W, b, dY, record=True)
    halves = LinearReluTrainStep(m, n, k, cuda_device, x_checkpoint="int8", **options)
    halves.forward(X, W, b)
    X.fill_(float("nan"))
    halves.backward(W, dY)
    torch.cuda.synchronize()
    assert set(events.phases) >= set(whole.PHASES)
    for name in ("Y", "mask", "dZ", "dX", "dW", "db", "Xq", "x_scale"):
        assert torch.equal(getattr(whole, name), getattr(halves, name)), name
