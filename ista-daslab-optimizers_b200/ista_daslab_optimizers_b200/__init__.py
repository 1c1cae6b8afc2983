"""B200-native MicroAdam optimizer step (drop-in for ista_daslab_optimizers.MicroAdam), and the distillation of a frozen 8-bit teacher into the
model it trains."""
from .distillation import distill_loss, distill_step, int8_matmul, quantize_rows, topk_logits
from .micro_adam import MicroAdam
from .tools import CopyDirection, block_split, get_first_device

__all__ = ['MicroAdam', 'CopyDirection', 'block_split', 'get_first_device', 'quantize_rows', 'int8_matmul', 'topk_logits', 'distill_loss',
           'distill_step']
