"""Serving: KV-cache generation for the Llama decoder (beyond the training-only reference)."""
from .controls import LogitControls, LogitProcessor
from .generator import ContinuousBatcher, Generator, Request

__all__ = ["ContinuousBatcher", "Generator", "LogitControls", "LogitProcessor", "Request"]
