"""fastlstm_b200 — B200 (sm_100a) LSTM layer behind the FastLSTM module surface.

The CUDA library (libfastlstm_b200.so, C ABI in include/fastlstm_b200.h) is
loaded on first use; there is no CPU or PyTorch fallback.
"""
from .language import (BeamStep, EightBitRows, TokenLogProbs, beam_step, dropout, embedding, reorder_states, rms_norm,
                       rms_norm_e4m3, token_log_probs)
from .lstm import (FastLSTM, PersistentLSTMfn, Wgrad, check_status, lstm_persistent_bwd,
                   lstm_persistent_fwd, persistent_lstm, plan_detail, plan_name)
from .optim import AdamW

__all__ = ["AdamW", "BeamStep", "EightBitRows", "FastLSTM", "PersistentLSTMfn", "TokenLogProbs", "Wgrad", "beam_step", "check_status",
           "dropout", "embedding", "lstm_persistent_bwd", "lstm_persistent_fwd", "persistent_lstm", "plan_detail", "plan_name",
           "reorder_states", "rms_norm", "rms_norm_e4m3", "token_log_probs"]
