"""What goes on behind a prompt pass: another prompt pass, and the default decoder's own loop (persistent local and global
steps, captured graphs). As in tests/test_prompt_gpu.py, the byte loop is no reference: both are compared with the fp32
decoder of the same weights over the same patch starts, and the prompt pass may be at most twice as far from it."""

import pytest
import torch
from test_prompt_gpu import SMALL, fed, text

from byteprof_b200 import _lib
from byteprof_b200.optim.bolmo_e2e import BolmoDecoder

pytestmark = pytest.mark.gpu
DEFAULT = dict(global_layers=2, max_patches=128)  # the other sizes and the fused steps are the default's


@pytest.mark.parametrize("cut", [1, 16, 33, 89])
def test_two_prefills_continue_each_other_whatever_the_flags_are(cut):
    ids = text(90, 3)
    two, loop, exact = BolmoDecoder(**SMALL), BolmoDecoder(**SMALL), BolmoDecoder(precision="fp32", **SMALL)
    first, f1, o1 = two.prefill(ids[:cut])
    second, f2, o2 = two.prefill(ids[cut:], first_patch=f1[-1])
    opened = o1 + o2
    assert opened[0] and opened[1:] == (f1 + f2)[:-1]
    assert two.patches == sum(opened) == int(two.pos)
    want, step = fed(exact, ids, opened), fed(loop, ids, opened)
    for part, got in ((slice(0, cut), first), (slice(cut, 90), second)):
        e_two, e_loop = (got.double() - want[part]).norm().item(), (step[part] - want[part]).norm().item()
        assert e_two <= 2 * e_loop, (part, e_two, e_loop)


@pytest.mark.parametrize("captured", [False, True])
def test_the_default_decoder_goes_on_behind_a_prompt(captured):
    ids = text(64, 13)
    n = 40
    dec, loop, exact = BolmoDecoder(**DEFAULT), BolmoDecoder(**DEFAULT), BolmoDecoder(precision="fp32", **DEFAULT)
    if captured:
        dec.capture()
    logits, flags, opened = dec.prefill(ids[:n])
    more = [flags[-1]] + [i % 3 != 1 for i in range(len(ids) - n - 1)]
    starts = opened + more
    want, step = fed(exact, ids, starts), fed(loop, ids, starts)
    assert (logits.double() - want[:n]).norm() <= 2 * (step[:n] - want[:n]).norm()
    if captured:
        rows = []
        for b, o in zip(ids[n:], more):
            tokens, _, fed_starts, _ = dec.steps(1, bytes_=[b], patches=[o])
            assert fed_starts == [o] and tokens == [int(dec.logits[0].argmax())]
            rows.append(dec.logits[0].double().clone())
        cont = torch.stack(rows)
    else:
        cont = fed(dec, ids[n:], more)
    assert (cont - want[n:]).norm() <= 2 * (step[n:] - want[n:]).norm()
    assert dec.patches == loop.patches and int(dec.pos) == int(loop.pos) and dec.parity == (1 + len(more)) % 2
    assert _lib.device_errors() == 0


def test_a_prompt_behind_the_captured_loop():
    """The loop first, then a prompt pass over the state that it left, then the loop again."""
    ids = text(60, 17)
    dec, loop, exact = BolmoDecoder(**DEFAULT), BolmoDecoder(**DEFAULT), BolmoDecoder(precision="fp32", **DEFAULT)
    dec.capture()
    head = [True] + [i % 4 != 2 for i in range(14)]
    got = [fed(dec, ids[:15], head)]
    logits, flags, opened = dec.prefill(ids[15:45], first_patch=False)
    got.append(logits.double())
    tail = [flags[-1]] + [i % 2 == 0 for i in range(14)]
    got.append(fed(dec, ids[45:], tail))
    starts = head + opened + tail
    want, step = fed(exact, ids, starts), fed(loop, ids, starts)
    for part, y in zip((slice(0, 15), slice(15, 45), slice(45, 60)), got):
        assert (y - want[part]).norm() <= 2 * (step[part] - want[part]).norm()
