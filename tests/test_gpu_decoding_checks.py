"""What the Python forms of the calls between projection and cache, and behind the logits, refuse: tensors of another device,
type, shape or order, before anything is launched; and that they go to the stream and device they are asked for."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_parity import pk  # noqa: E402, F401

pytestmark = pytest.mark.gpu

f16, f32, i32, u8 = torch.float16, torch.float32, torch.int32, torch.uint8


def t(*shape, kind=f16):
    return torch.zeros(shape, dtype=kind, device="cuda")


def calls(pk):  # noqa: F811
    """name -> (call, arguments that are all right)."""
    words = pk.rotary_frequencies(32)
    heads = dict(query=t(5, 4, 64), key=t(5, 2, 64), query_weight=t(64), key_weight=t(64), positions=t(5, kind=i32), frequencies=words)
    return {
        "head_norm_rotary": (pk.head_norm_rotary, {**heads, "query_out": t(5, 4, 64), "key_out": t(5, 2, 64)}),
        "head_norm_rotary_write": (pk.head_norm_rotary_write, {
            **heads, "value": t(5, 2, 64), "slots": torch.arange(5, dtype=i32, device="cuda"), "query_out": t(5, 4, 64), "key_cache": t(3, 2, 16, 64),
            "value_cache": t(3, 2, 64, 16)}),
        "beam_select": (lambda **kw: pk.beam_select(**kw, end_token=1), dict(
            logits=t(2, 3, 50), scores=t(2, 3, kind=f32), ended=t(2, 3, kind=torch.bool), out_scores=t(2, 4, kind=f32), out_tokens=t(2, 4, kind=i32),
            out_parents=t(2, 4, kind=i32), out_ended=t(2, 4, kind=torch.bool), workspace=t(pk.beam_select_workspace_bytes(2, 3, 50, 4), kind=u8))),
        "beam_reorder": (pk.beam_reorder, dict(state=t(2, 3, 8), parents=t(2, 3, kind=i32), output=t(2, 3, 8))),
        "page_fork": (lambda **kw: pk.page_fork(**kw, page_size=16), dict(
            parents=t(3, kind=i32), block_table=t(3, 4, kind=i32), lengths=t(3, kind=i32), free_pages=t(9, kind=i32), free_range=t(2, kind=i32),
            new_table=t(3, 4, kind=i32), new_lengths=t(3, kind=i32), copies=t(3, 2, kind=i32), freed=t(20, kind=i32), info=t(4, kind=i32),
            workspace=t(pk.page_fork_workspace_bytes(3, 4, 20), kind=u8), held=t(20, kind=u8))),
        "page_keep": (pk.page_keep, dict(info=t(4, kind=i32), freed=t(20, kind=i32), free_pages=t(9, kind=i32), free_range=t(2, kind=i32))),
        "paged_cache_copy": (pk.paged_cache_copy, dict(copies=t(3, 2, kind=i32), key_cache=t(3, 2, 16, 64), value_cache=t(3, 2, 64, 16))),
    }


NAMES = ["head_norm_rotary", "head_norm_rotary_write", "beam_select", "beam_reorder", "page_fork", "page_keep", "paged_cache_copy"]


@pytest.mark.parametrize("name", NAMES)
def test_each_tensor_is_checked(pk, name):  # noqa: F811
    call, right = calls(pk)[name]
    call(**right)
    for arg, x in right.items():
        wrong = [("cpu", x.cpu()), ("type", x.double())]
        if arg != "workspace":  # (its length is the library's to check)
            longer = torch.zeros((x.shape[0] + 1,) + tuple(x.shape[1:]), dtype=x.dtype, device="cuda")
            if arg not in ("free_pages", "freed", "frequencies", "copies") or (name, arg) == ("page_fork", "copies"):
                wrong.append(("shape", longer))
        spread = torch.zeros(tuple(x.shape) + (2,), dtype=x.dtype, device="cuda")[..., 0]
        wrong.append(("order", spread))
        for what, bad in wrong:
            with pytest.raises((ValueError, pk.PkError)):
                call(**{**right, arg: bad})
                pytest.fail(f"{name}: {arg} of another {what} was taken")
    torch.cuda.synchronize()


@pytest.mark.parametrize("name,arg", [("head_norm_rotary", "key_out"), ("head_norm_rotary", "key"), ("head_norm_rotary", "positions"),
                                      ("head_norm_rotary_write", "positions")])
def test_halves_of_a_call_are_refused(pk, name, arg):  # noqa: F811
    call, right = calls(pk)[name]
    with pytest.raises(ValueError):
        call(**{**right, arg: None})


def test_small_workspaces_are_refused(pk):  # noqa: F811
    for name in ("beam_select", "page_fork"):
        call, right = calls(pk)[name]
        with pytest.raises(pk.PkError):
            call(**{**right, "workspace": right["workspace"][:-1].clone()})


def test_an_end_token_beyond_the_vocabulary(pk):  # noqa: F811
    _, right = calls(pk)["beam_select"]
    for end in (50, -1, 1 << 31, (1 << 32) + 1):  # (ended beams need one)
        with pytest.raises((ValueError, pk.PkError)):
            pk.beam_select(**right, end_token=end)


@pytest.mark.parametrize("name", NAMES)
def test_calls_are_captured_on_their_stream(pk, name):  # noqa: F811
    """Whatever stream is current, a call on a named one is recorded there."""
    call, right = calls(pk)[name]
    call(**right)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(**right)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
