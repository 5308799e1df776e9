"""Where a kernel's error word is read: ahead of a trainer's update, and at the end of generation and beam search, with the text of the kernel that set it."""
import pytest
import torch

from linear_moe_b200.infer import generation as G
from linear_moe_b200.ops import gemm
from linear_moe_b200.parallel import fused_comm
from test_softmax_layers import EOD, model, prompts


@pytest.fixture
def words(monkeypatch):
    """The status tensor, its error word, and a word of another device."""
    status, other = torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(fused_comm, "STATUS", status)
    monkeypatch.setattr(gemm, "_ERR", status[1:2])
    monkeypatch.setattr(gemm, "OTHER_WORDS", [other])
    return status[1:2], other


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("code,text", [(0x12000, "page number outside the pool"), (0x14001, "one-token attention: a bounded wait"), (0x26700, "attention with key ranges"), (0x31, "GEMM")])
def test_the_trainer_says_which_kernel(words, which, code, text):
    words[which][0] = code
    with pytest.raises(RuntimeError, match=text + r".*0x%x.*iteration 7" % code):
        fused_comm.check_status("iteration 7")
    fused_comm.check_status()                                  # read once
    gemm.check_error()


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("paged", [False, True])
def test_generation_reads_the_words(words, which, paged):
    m = model(num_layers=1)
    base, lengths = prompts(L=14)
    G.generate_tokens(m, base.clone(), lengths, top_k=1, paged=paged)
    words[which][0] = 0x12000
    with pytest.raises(RuntimeError, match="page number outside the pool"):
        G.generate_tokens(m, base.clone(), lengths, top_k=1, paged=paged)
    words[which][0] = 0x13000
    with pytest.raises(RuntimeError, match="a row that is none"):
        G.beam_search(m, base[:1, :9], 2, 3, EOD, paged=paged)
    G.beam_search(m, base[:1, :9], 2, 3, EOD, paged=paged)


@pytest.mark.parametrize("other", [False, True])
def test_words_made_under_inference_mode(monkeypatch, other):
    """The first kernel of a process may run there; the check that finds its error may not."""
    from linear_moe_b200.ops import cuda as K
    monkeypatch.setattr(fused_comm, "STATUS", None)
    monkeypatch.setattr(gemm, "_ERR", None)
    monkeypatch.setattr(gemm, "OTHER_WORDS", [])
    monkeypatch.setattr(K, "_ERROR_WORDS", {})
    cpu = torch.device("cpu")
    with torch.inference_mode():
        if other:
            gemm._err(torch.device("meta"))                    # the status tensor lies elsewhere
        K.error_word(cpu)
    word = K._ERROR_WORDS[cpu]
    if other:
        monkeypatch.setattr(gemm, "_ERR", None)
        assert len(gemm.OTHER_WORDS) == 1
    for _ in range(2):
        word.data[0] = 0x13000
        with pytest.raises(RuntimeError, match="a row that is none"):
            gemm.check_error()
        assert int(word) == 0
