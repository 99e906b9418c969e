//go:build linux && amd64

package cgo_bridge

// Wrappers for the operators at the two ends of a language model's training step: embedding lookup and its gradient,
// dropout, and the linear cross entropy with its gradients.  Buffers and workspaces are handles as everywhere in this
// package; work runs on the library's stream, like the optimizer steps that take the gradients.

/*
#include <stdint.h>
#include "gometal_hip.h"
*/
import "C"

import (
	"fmt"
	"runtime"
	"unsafe"
)

// Element types of the operators (memory/tensor.go:12-17, and bfloat16).
const (
	LMFloat32  = 0
	LMFloat16  = 2
	LMBFloat16 = 4
)

// lastError is the message of the last call on this OS thread (where the library keeps it).
func lastError() string {
	var text []byte
	for at := (*byte)(unsafe.Pointer(C.gm_last_error())); at != nil && *at != 0; at = (*byte)(unsafe.Add(unsafe.Pointer(at), 1)) {
		text = append(text, *at)
	}
	return string(text)
}

// lmCall makes a call and turns its code into an error that says what the library says: the workspace that is needed, the size
// or handle that is wrong.
func lmCall(what string, call func() C.int) error {
	runtime.LockOSThread()
	defer runtime.UnlockOSThread()
	if rc := call(); rc != 0 {
		return fmt.Errorf("%s failed with error code: %d: %s", what, int(rc), lastError())
	}
	return nil
}

func lmFlag(b bool) int {
	if b {
		return 1
	}
	return 0
}

// AllocateWorkspace allocates a buffer of any length (AllocateMetalBuffer's size is an int32 in C).  Freed with
// DeallocateMetalBuffer.
func AllocateWorkspace(device unsafe.Pointer, bytes uint64) (unsafe.Pointer, error) {
	runtime.LockOSThread()
	defer runtime.UnlockOSThread()
	buffer := C.gm_allocate_workspace(C.uintptr_t(uintptr(device)), C.uintptr_t(uintptr(bytes)))
	if buffer == 0 {
		return nil, fmt.Errorf("failed to allocate workspace of size %d: %s", bytes, lastError())
	}
	return unsafe.Pointer(uintptr(buffer)), nil
}

// Dropout writes input / (1 - probability) where the generator keeps an element and 0 elsewhere, plus the residual
// (nil: none).  The backward pass is the same call on the gradient.
func Dropout(device, input, residual, output unsafe.Pointer, numElements, dataType int, probability float32, rngState unsafe.Pointer, site int) error {
	return lmCall("dropout", func() C.int {
		return C.execute_dropout(
			C.uintptr_t(uintptr(device)), C.uintptr_t(0), C.uintptr_t(uintptr(input)), C.uintptr_t(uintptr(residual)), C.uintptr_t(uintptr(output)),
			C.int(numElements), C.int(dataType), C.float(probability), C.uintptr_t(uintptr(rngState)), C.int(site),
		)
	})
}

// AdvanceRNGState moves dropout's generator state to the next training step.
func AdvanceRNGState(device, rngState unsafe.Pointer) error {
	return lmCall("generator state", func() C.int {
		return C.gm_rng_state_advance(C.uintptr_t(uintptr(device)), C.uintptr_t(0), C.uintptr_t(uintptr(rngState)))
	})
}

// EmbeddingLookup gathers scaled rows of the table, with dropout if the probability is above 0; tokens outside the
// vocabulary give rows of zeros.
func EmbeddingLookup(device, table, tokens, output unsafe.Pointer, numTokens, vocabSize, dim, tableStride, outputStride, dataType int,
	scale, dropoutProbability float32, rngState unsafe.Pointer, dropoutSite int) error {
	return lmCall("embedding lookup", func() C.int {
		return C.execute_embedding_lookup(
			C.uintptr_t(uintptr(device)), C.uintptr_t(0), C.uintptr_t(uintptr(table)), C.uintptr_t(uintptr(tokens)), C.uintptr_t(uintptr(output)),
			C.int(numTokens), C.int(vocabSize), C.int(dim), C.int(tableStride), C.int(outputStride), C.int(dataType),
			C.float(scale), C.float(dropoutProbability), C.uintptr_t(uintptr(rngState)), C.int(dropoutSite),
		)
	})
}

// EmbeddingGradientWorkspace returns the bytes that EmbeddingGradient needs.
func EmbeddingGradientWorkspace(numTokens, vocabSize, dim int) uint64 {
	return uint64(C.gm_embedding_gradient_workspace(C.int(numTokens), C.int(vocabSize), C.int(dim)))
}

// EmbeddingGradient writes (accumulate: adds) the lookup's gradient into the table's gradient, summed per word over the
// positions in their order.
func EmbeddingGradient(device, outputGradient, tokens, tableGradient unsafe.Pointer,
	numTokens, vocabSize, dim, outputGradientStride, tableGradientStride, dataType, gradientType int, scale float32, paddingToken int,
	accumulate bool, dropoutProbability float32, rngState unsafe.Pointer, dropoutSite int, workspace unsafe.Pointer, workspaceBytes uint64) error {
	return lmCall("embedding gradient", func() C.int {
		return C.execute_embedding_gradient(
			C.uintptr_t(uintptr(device)), C.uintptr_t(0), C.uintptr_t(uintptr(outputGradient)), C.uintptr_t(uintptr(tokens)),
			C.uintptr_t(uintptr(tableGradient)), C.int(numTokens), C.int(vocabSize), C.int(dim), C.int(outputGradientStride),
			C.int(tableGradientStride), C.int(dataType), C.int(gradientType), C.float(scale), C.int(paddingToken), C.int(lmFlag(accumulate)),
			C.float(dropoutProbability), C.uintptr_t(uintptr(rngState)), C.int(dropoutSite), C.uintptr_t(uintptr(workspace)),
			C.uintptr_t(uintptr(workspaceBytes)),
		)
	})
}

// LinearCrossEntropyWorkspace returns the bytes for the fastest form of LinearCrossEntropy over these weights.
func LinearCrossEntropyWorkspace(numTokens, vocabSize, dim int, weight unsafe.Pointer, weightStride, dataType, gradientType int, withGradients bool) uint64 {
	return uint64(C.gm_linear_cross_entropy_workspace(C.int(numTokens), C.int(vocabSize), C.int(dim), C.uintptr_t(uintptr(weight)),
		C.int(weightStride), C.int(dataType), C.int(gradientType), C.int(lmFlag(withGradients))))
}

// LinearCrossEntropyLeastWorkspace returns the fewest bytes that LinearCrossEntropy works with.
func LinearCrossEntropyLeastWorkspace(numTokens, vocabSize, dim int, weight unsafe.Pointer, weightStride, dataType, gradientType int, withGradients bool) uint64 {
	return uint64(C.gm_linear_cross_entropy_least_workspace(C.int(numTokens), C.int(vocabSize), C.int(dim), C.uintptr_t(uintptr(weight)),
		C.int(weightStride), C.int(dataType), C.int(gradientType), C.int(lmFlag(withGradients))))
}

// LinearCrossEntropy computes the softmax cross entropy of hidden * weight^T (losses: one per token; loss: their mean or sum
// and the number of tokens that count) and, where the handles are not nil, its gradients times gradientScale times the
// loss scale of ampState.
func LinearCrossEntropy(device, hidden, weight, targets, losses, loss, hiddenGradient, weightGradient unsafe.Pointer,
	numTokens, vocabSize, dim, hiddenStride, weightStride, hiddenGradientStride, weightGradientStride, dataType, gradientType, ignoreIndex int,
	mean bool, gradientScale float32, ampState unsafe.Pointer, accumulate bool, workspace unsafe.Pointer, workspaceBytes uint64) error {
	return lmCall("linear cross entropy", func() C.int {
		return C.execute_linear_cross_entropy(
			C.uintptr_t(uintptr(device)), C.uintptr_t(0), C.uintptr_t(uintptr(hidden)), C.uintptr_t(uintptr(weight)), C.uintptr_t(uintptr(targets)),
			C.uintptr_t(uintptr(losses)), C.uintptr_t(uintptr(loss)), C.uintptr_t(uintptr(hiddenGradient)), C.uintptr_t(uintptr(weightGradient)),
			C.int(numTokens), C.int(vocabSize), C.int(dim), C.int(hiddenStride), C.int(weightStride), C.int(hiddenGradientStride),
			C.int(weightGradientStride), C.int(dataType), C.int(gradientType), C.int(ignoreIndex), C.int(lmFlag(mean)), C.float(gradientScale),
			C.uintptr_t(uintptr(ampState)), C.int(lmFlag(accumulate)), C.uintptr_t(uintptr(workspace)), C.uintptr_t(uintptr(workspaceBytes)),
		)
	})
}
