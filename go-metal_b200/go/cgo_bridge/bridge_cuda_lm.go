//go:build cuda

package cgo_bridge

/*
#include "gometal_cuda.h"
*/
import "C"

import (
	"fmt"
	"unsafe"
)

// Operators at the two ends of a language model, with no counterpart in the Metal build:
// token embedding, dropout, and softmax cross entropy over a vocabulary, each with its
// gradient.  All run on the device's stream and return without waiting; workspaces are the
// caller's and hold nothing between calls.

// DType is an element type of these operators: the codes of memory.DataType, and BFloat16.
type DType int

const (
	Float32  DType = 0
	Float16  DType = 2
	BFloat16 DType = 4
)

// Dropout describes the counter-based mask.  A use of its own (layer, step) takes an Offset of
// its own; OffsetDevice, if set, is the device address of a uint64 added to it.
type Dropout struct {
	P            float32
	Seed, Offset uint64
	OffsetDevice unsafe.Pointer
}

func (d *Dropout) c() *C.gm_dropout_t {
	if d == nil {
		return nil
	}
	out := new(C.gm_dropout_t)
	out.p, out.seed, out.offset = C.float(d.P), C.uint64_t(d.Seed), C.uint64_t(d.Offset)
	out.offset_device = handle(d.OffsetDevice)
	return out
}

// DropoutAsync sets y = residual + dropout(x); residual may be nil.  The backward pass is the
// same call on the gradient without a residual.  Strides are in elements.
func DropoutAsync(device unsafe.Pointer, dtype DType, rows, cols int64, x unsafe.Pointer, ldX int64, residual unsafe.Pointer, ldResidual int64,
	y unsafe.Pointer, ldY int64, d Dropout) error {
	return stepError("dropout", C.gm_dropout_async(handle(device), C.int(dtype), C.int64_t(rows), C.int64_t(cols), handle(x), C.int64_t(ldX),
		handle(residual), C.int64_t(ldResidual), handle(y), C.int64_t(ldY), d.c()))
}

// Embedding is a lookup of Tokens rows of Dim columns in a table of Vocab rows, times Scale.
type Embedding struct {
	DType              DType
	Tokens, Dim, Vocab int64
	LdTable, LdOut     int64
	PaddingToken       int64 // its row takes no gradient; -1: none
	Scale              float32
}

func (e Embedding) c() *C.gm_embedding_t {
	out := new(C.gm_embedding_t)
	out.dtype = C.int(e.DType)
	out.tokens, out.dim, out.vocab = C.int64_t(e.Tokens), C.int64_t(e.Dim), C.int64_t(e.Vocab)
	out.ld_table, out.ld_out = C.int64_t(e.LdTable), C.int64_t(e.LdOut)
	out.padding_token, out.scale = C.int64_t(e.PaddingToken), C.float(e.Scale)
	return out
}

// ForwardAsync sets out[t] = dropout(scale * table[tokens[t]]); d may be nil.
func (e Embedding) ForwardAsync(device, table, tokens, out unsafe.Pointer, d *Dropout) error {
	return stepError("embedding", C.gm_embedding_forward_async(handle(device), e.c(), handle(table), handle(tokens), handle(out), d.c()))
}

// WorkspaceBytes is what BackwardAsync needs.
func (e Embedding) WorkspaceBytes() (int64, error) {
	n := int64(C.gm_embedding_workspace_bytes(e.c()))
	if n < 0 {
		return 0, fmt.Errorf("embedding: %s", lastError())
	}
	return n, nil
}

// BackwardAsync writes the table's gradient (accumulate: adds to the rows that tokens point at).
func (e Embedding) BackwardAsync(device, tokens, dout unsafe.Pointer, d *Dropout, dtable unsafe.Pointer, gradType DType, accumulate bool,
	workspace unsafe.Pointer, workspaceBytes int64) error {
	return stepError("embedding gradient", C.gm_embedding_backward_async(handle(device), e.c(), handle(tokens), handle(dout), d.c(), handle(dtable),
		C.int(gradType), cbool(accumulate), handle(workspace), C.int64_t(workspaceBytes)))
}

// LinearXent is the softmax cross entropy of Tokens hidden states of Dim columns over the Vocab
// rows of a table, without the logits in memory.
type LinearXent struct {
	DType              DType // Float16 or BFloat16
	Tokens, Dim, Vocab int64
	LdHidden, LdWeight int64
	Mean               bool
}

func (x LinearXent) c() *C.gm_linear_xent_t {
	out := new(C.gm_linear_xent_t)
	out.dtype = C.int(x.DType)
	out.tokens, out.dim, out.vocab = C.int64_t(x.Tokens), C.int64_t(x.Dim), C.int64_t(x.Vocab)
	out.ld_hidden, out.ld_weight = C.int64_t(x.LdHidden), C.int64_t(x.LdWeight)
	out.mean = cbool(x.Mean)
	return out
}

// WorkspaceBytes: pass 0 for the forward pass, 1 for both, 2 for the least the backward pass takes.
func (x LinearXent) WorkspaceBytes(pass int) (int64, error) {
	n := int64(C.gm_linear_xent_workspace_bytes(x.c(), C.int(pass)))
	if n < 0 {
		return 0, fmt.Errorf("vocabulary loss: %s", lastError())
	}
	return n, nil
}

// ForwardAsync writes a loss and a log-sum-exp per row and {loss, rows with a target} to total.
func (x LinearXent) ForwardAsync(device, hidden, weight, targets, losses, lse, total, workspace unsafe.Pointer, workspaceBytes int64) error {
	return stepError("vocabulary loss", C.gm_linear_xent_forward_async(handle(device), x.c(), handle(hidden), handle(weight), handle(targets),
		handle(losses), handle(lse), handle(total), handle(workspace), C.int64_t(workspaceBytes)))
}

// BackwardAsync writes both gradients (either may be nil), times gradScale and the float at
// scaleDevice (nil: 1), for which MixedAdam.StateDevicePtr is made.
func (x LinearXent) BackwardAsync(device, hidden, weight, targets, lse, scaleDevice unsafe.Pointer, gradScale float32, dHidden, dWeight unsafe.Pointer,
	accumulateWeight bool, workspace unsafe.Pointer, workspaceBytes int64) error {
	return stepError("vocabulary loss gradient", C.gm_linear_xent_backward_async(handle(device), x.c(), handle(hidden), handle(weight), handle(targets),
		handle(lse), handle(scaleDevice), C.float(gradScale), handle(dHidden), handle(dWeight), cbool(accumulateWeight), handle(workspace),
		C.int64_t(workspaceBytes)))
}

// LinearXentStatus waits for the device and reports a bounded wait of these products that ran out.
func LinearXentStatus(device unsafe.Pointer) error {
	return stepError("vocabulary loss", C.gm_linear_xent_status(handle(device)))
}

// StateDevicePtr is the device address of the loss-scale state, whose first member is the scale.
func (m *MixedAdam) StateDevicePtr() unsafe.Pointer {
	return unsafe.Pointer(uintptr(C.gm_mixed_state_device_ptr(m.h)))
}

func cbool(b bool) C.int {
	if b {
		return 1
	}
	return 0
}
