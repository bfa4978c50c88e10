from .batch import BatchStager, StepBatch, layout_step
from .engine import Engine
from .model import DecoderModel, expected_tensors
from .generate import GenerationResult, generate, plan_batches
from .beam import BeamResult, Hypothesis, generate_beams, plan_beam_batches

__all__ = ["BatchStager", "StepBatch", "layout_step", "Engine", "DecoderModel",
           "expected_tensors", "GenerationResult", "generate", "plan_batches",
           "BeamResult", "Hypothesis", "generate_beams", "plan_beam_batches"]
