"""What Muon's callers see of a wait that ran out: the error is recorded from the host, as such a wait records it."""
import pytest
import torch

from test_muon_gpu import matrix, optimizer

pytestmark = pytest.mark.gpu


@pytest.fixture
def failing():
    """Records an error; cleared at the end."""
    from d1._lib import check, library
    from d1.muon import muon_error

    def record(code=3):
        torch.cuda.synchronize()
        check(library().d1_muon_set_error(code))
    assert muon_error() == 0
    yield record
    muon_error()


SHAPES = [[(300, 200), (64, 90)], [(100, 120), (30, 40)], [(1024, 1024)] * 4]  # by single CTAs, in one launch, by pairs


@pytest.mark.parametrize('shapes', SHAPES)
def test_the_next_call_raises(shapes, failing):
    from d1._lib import D1Error
    from d1.muon import muon_error, orthogonalize
    opt, params, grads, copies = optimizer(shapes, lr=0.05)
    opt.step()
    opt.check()
    before = [t.clone() for t in params + copies + [opt.momentum]]
    failing()
    for _ in range(2):
        with pytest.raises(D1Error):
            opt.step()
    with pytest.raises(D1Error):
        orthogonalize(params[0])
    assert all(torch.equal(t, b) for t, b in zip(params + copies + [opt.momentum], before))
    assert muon_error() == 3 and muon_error() == 0
    opt.step()
    assert not torch.equal(params[0], before[0])
    orthogonalize(params[0])
    failing(5)
    with pytest.raises(D1Error):
        opt.check()
    opt.check()


@pytest.mark.parametrize('shapes', SHAPES)
def test_a_step_after_the_failure_changes_no_parameter(shapes, failing):
    """A captured step is replayed without a look at the error; the kernels look."""
    from d1.muon import muon_error
    opt, params, grads, copies = optimizer(shapes, lr=0.05)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    before = [t.clone() for t in params + copies]
    failing(4)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(t, b) for t, b in zip(params + copies, before))
    assert muon_error() == 4
    graph.replay()
    torch.cuda.synchronize()
    assert all(not torch.equal(t, b) for t, b in zip(params + copies, before)) and muon_error() == 0


def test_the_recurrent_head_raises(failing):
    from d1._lib import D1Error
    from d1.recurrent import RecurrentHead
    head = RecurrentHead(seed=2)
    g = torch.Generator(device='cuda').manual_seed(0)
    h = torch.randn(2, 16, 512, device='cuda', generator=g).to(torch.bfloat16)
    joint = torch.zeros(2, 16, dtype=torch.int64, device='cuda')
    legal = torch.full((2, 16), 0x7fffffff, dtype=torch.int32, device='cuda')
    old, adv = torch.full((2, 16), -3.0, device='cuda'), torch.ones(2, 16, device='cuda')
    head.update(h, joint, legal, old, adv, head.state(16))
    before = {k: p.clone() for k, p in head.params.items()}
    failing()
    with pytest.raises(D1Error):
        head.update(h, joint, legal, old, adv, head.state(16))
    assert all(torch.equal(p, before[k]) for k, p in head.params.items())


def test_first_call_in_a_capture():
    """Nothing is allocated while a graph is captured, in a process whose first call that is."""
    import pathlib
    import subprocess
    import sys
    code = ('import torch\nfrom d1.muon import orthogonalize\nx = torch.randn(100, 80, device="cuda")\ng = torch.cuda.CUDAGraph()\n'
            'with torch.cuda.graph(g):\n    y = orthogonalize(x)\ng.replay()\ntorch.cuda.synchronize()\nassert torch.equal(y, orthogonalize(x))\nprint("ok")')
    root = pathlib.Path(__file__).resolve().parents[1] / 'dcss-auto_b200'
    r = subprocess.run([sys.executable, '-c', code], capture_output=True, text=True, env={**__import__('os').environ, 'PYTHONPATH': str(root)}, timeout=300)
    assert r.stdout == 'ok\n', r.stderr


def test_with_another_default_device():
    """The word in host memory is one whatever torch's default device is, in a process whose first call that is."""
    import os
    import pathlib
    import subprocess
    import sys
    code = ('import torch\nfrom d1.muon import orthogonalize\ntorch.set_default_device("cuda")\nx = torch.randn(100, 80)\ny = orthogonalize(x)\n'
            'assert torch.equal(y, orthogonalize(x))\nprint("ok")')
    root = pathlib.Path(__file__).resolve().parents[1] / 'dcss-auto_b200'
    r = subprocess.run([sys.executable, '-c', code], capture_output=True, text=True, env={**os.environ, 'PYTHONPATH': str(root)}, timeout=300)
    assert r.stdout == 'ok\n', r.stderr
